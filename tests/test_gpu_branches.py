"""GPU tests of keep_drafts and fork_sequences against the restatements in
branch_reference.py. Rows, tables, counts and lists are compared exactly."""
import numpy as np
import pytest

import branch_reference as ref
import sgl_rocm_kv as kv
from branch_reference import NONE
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


class Bytes:
    """A pool of bytes with all layers, `widths` bytes a token and tensor in `heads` chunks, token- or head-major, `shift`
    bytes into its allocation; `gap` bytes lie between its regions and pages."""

    def __init__(self, rng, *, page, pages, layers, heads, widths, hnd=False, shift=0, gap=0):
        self.page, self.pages, self.layers, self.heads, self.widths, self.hnd, self.shift = page, pages, layers, heads, widths, hnd, shift
        self.layer_stride = page * sum(widths) + gap
        self.page_stride = layers * self.layer_stride + gap
        self.raw = rng.integers(0, 256, shift + pages * self.page_stride, dtype=np.uint8)
        self.device = hip.DeviceBuffer.from_array(self.raw)

    def view(self):
        offsets = (0, self.page * self.widths[0])
        return kv.pool_view(self.device.ptr + self.shift, self.device.nbytes - self.shift, page_size=self.page,
                            page_stride_bytes=self.page_stride, page_count=self.pages,
                            tensor_offset=offsets[:len(self.widths)], row_bytes=self.widths[0],
                            tensor_count=len(self.widths), heads=self.heads, head_layout=kv.HND if self.hnd else kv.NHD,
                            value_row_bytes=self.widths[1] if len(self.widths) == 2 and self.widths[1] != self.widths[0] else 0)

    def region(self, raw, page, layer, tensor):
        """[position][head][bytes] of a page's tensor: a view."""
        at = self.shift + page * self.page_stride + layer * self.layer_stride + self.page * sum(self.widths[:tensor])
        flat = raw[at:at + self.page * self.widths[tensor]]
        chunk = self.widths[tensor] // self.heads
        if self.hnd:
            return flat.reshape(self.heads, self.page, chunk).transpose(1, 0, 2)
        return flat.reshape(self.page, self.heads, chunk)

    def move(self, to_raw, to, from_raw, source, rows=1):
        """Rows from slot `source` on to slot `to` on (of one page each), every layer and tensor."""
        for layer in range(self.layers):
            for t in range(len(self.widths)):
                a, b = self.region(to_raw, int(to) // self.page, layer, t), self.region(from_raw, int(source) // self.page, layer, t)
                i, j = int(to) % self.page, int(source) % self.page
                a[i:i + rows] = b[j:j + rows]

    def call(self):
        return dict(layer_count=self.layers, layer_stride_bytes=self.layer_stride)


POOLS = [
    dict(page=16, layers=3, heads=8, widths=(2048, 2048)),
    dict(page=16, layers=2, heads=2, widths=(256, 256), hnd=True),
    dict(page=64, layers=2, heads=1, widths=(1152, 1024)),                 # a pair of unequal widths
    dict(page=64, layers=2, heads=1, widths=(649,)),                       # packed rows of an odd width
    dict(page=7, layers=3, heads=3, widths=(30, 18), gap=2),
    dict(page=16, layers=1, heads=4, widths=(64, 64), hnd=True, shift=4),
    dict(page=5, layers=2, heads=2, widths=(34, 34), hnd=True, shift=1),
    dict(page=1, layers=4, heads=2, widths=(128, 128)),
    dict(page=32, layers=2, heads=8, widths=(5120, 5120), gap=16),         # rows of more pieces than a workgroup's threads
]


def _ids(p):
    return "-".join(f"{a}{b}" for a, b in p.items()).replace(" ", "")


# ---- keep_drafts ----------------------------------------------------------------------------


class Drafts:
    def __init__(self, rng, pool, contexts, drafts, kept, max_kept):
        self.pool, self.contexts = pool, list(contexts)
        lengths = [c + n for c, n in zip(contexts, drafts)]
        need = [-(-n // pool.page) for n in lengths]
        assert sum(need) <= pool.pages
        pages, at, slots, self.offsets = rng.permutation(pool.pages), 0, [], [0]
        for n, c in zip(lengths, need):
            slots.append((pages[at:at + c, None] * pool.page + np.arange(pool.page)).reshape(-1)[:n])
            self.offsets.append(self.offsets[-1] + n)
            at += c
        self.slots = np.concatenate(slots).astype(np.uint64)
        self.lists = np.full((len(lengths), max_kept), NONE, np.uint32)
        for r, own in enumerate(kept):
            self.lists[r, :len(own)] = own

    def run(self, k, stream=None):
        plan = kv.DraftPlan.new(request_count=len(self.contexts), sequence_slot_count=len(self.slots),
                                max_kept=self.lists.shape[1])
        self.given = dict(request_lengths=hip.DeviceBuffer.from_array(np.asarray(self.contexts, np.uint64)),
                          request_slot_offsets=hip.DeviceBuffer.from_array(np.asarray(self.offsets, np.uint64)),
                          sequence_slots=hip.DeviceBuffer.from_array(self.slots), kept=hip.DeviceBuffer.from_array(self.lists))
        k.keep_drafts(plan, kv.DraftBuffers(**self.given), self.pool.view(), stream=stream, **self.pool.call())
        hip.synchronize()
        return self.pool.device.download()

    def want(self, skip=()):
        out = self.pool.raw.copy()
        for r, own in enumerate(self.lists):
            if r in skip:
                continue
            at = int(self.offsets[r]) + self.contexts[r]
            for i, draft in enumerate(own[own != NONE]):
                self.pool.move(out, self.slots[at + i], self.pool.raw, self.slots[at + int(draft)])
        return out


@pytest.mark.parametrize("shape", POOLS, ids=_ids)
def test_kept_rows(k, shape):
    rng = np.random.default_rng(11)
    contexts, drafts = (20, 0, 33, 1, 7), (24, 9, 40, 1, 16)
    kept = [sorted(rng.choice(n, size, replace=False)) for n, size in zip(drafts, (9, 9, 11, 1, 0))]
    kept[2] = list(range(29, 40))  # all moved, over each other's places
    pool = Bytes(rng, pages=sum(-(-(c + n) // shape["page"]) for c, n in zip(contexts, drafts)) + 3, **shape)
    case = Drafts(rng, pool, contexts, drafts, kept, 12)
    _say(f"keep_drafts {shape}")
    got = case.run(k)
    k.check_errors()
    assert np.array_equal(got, case.want())


def test_long_lists_move_over_themselves(k):
    """Hundreds of rows, each moved by one or two places: every row is read before its place is written to."""
    rng = np.random.default_rng(12)
    pool = Bytes(rng, page=16, pages=130, layers=2, heads=2, widths=(64, 64))
    kept = [np.arange(1, 900), np.delete(np.arange(700), [3, 300])]
    case = Drafts(rng, pool, (5, 0), (901, 700), kept, 1000)
    got = case.run(k)
    k.check_errors()
    assert np.array_equal(got, case.want())


def test_nothing_to_move(k):
    rng = np.random.default_rng(13)
    pool = Bytes(rng, page=16, pages=9, layers=2, heads=2, widths=(64, 64))
    case = Drafts(rng, pool, (5, 0), (12, 7), [range(12), ()], 12)
    case.slots[0] = 2 ** 63  # a context slot: not looked at
    case.slots[5 + 11] = 2 ** 63  # stays where it is
    got = case.run(k)
    k.check_errors()
    assert np.array_equal(got, pool.raw)


@pytest.mark.parametrize("what,flags", [("order", 2), ("twice", 2), ("past", 2), ("hole", 2), ("range", 2), ("length", 2),
                                        ("source", 4), ("destination", 4)])
def test_a_bad_request_is_left_as_it_is(k, what, flags):
    rng = np.random.default_rng(14)
    pool = Bytes(rng, page=16, pages=12, layers=2, heads=2, widths=(64, 64))
    case = Drafts(rng, pool, (5, 9, 3), (12, 17, 8), [(1, 4, 5), (2, 3, 9, 16), (0, 7)], 5)
    at = case.offsets[1] + 9
    if what == "order":
        case.lists[1, 1:3] = (9, 3)
    elif what == "twice":
        case.lists[1, 2] = 3
    elif what == "past":
        case.lists[1, 3] = 17
    elif what == "hole":
        case.lists[1, 1] = NONE
    elif what == "range":
        case.offsets[1:3] = case.offsets[2], case.offsets[1]
    elif what == "length":
        case.contexts[1] = 2 ** 63
    elif what == "source":
        case.slots[at + 9] = 12 * 16
    elif what == "destination":
        case.slots[at] = 2 ** 40
    if what == "range":  # the neighbours' ranges change with it
        case.lists[0] = case.lists[2] = NONE
    got = case.run(k)
    with pytest.raises(kv.KvError) as e:
        k.check_errors()
    assert (e.value.variant, e.value.fields[0]) == ("DeviceMetadataInvalid", flags)
    assert np.array_equal(got, case.want(skip=(1,)))
    k.check_errors()


def test_keep_refusals(k):
    rng = np.random.default_rng(15)
    pool = Bytes(rng, page=16, pages=12, layers=2, heads=2, widths=(64, 64))
    case = Drafts(rng, pool, (5, 9), (12, 17), [(1, 4), (2,)], 2)
    case.run(k)
    plan = kv.DraftPlan.new(request_count=2, sequence_slot_count=len(case.slots), max_kept=2)

    def refused(variant, name, view=None, layers=2, stride=pool.layer_stride, **change):
        with pytest.raises(kv.KvError) as e:
            k.keep_drafts(plan, kv.DraftBuffers(**{**case.given, **change}), pool.view() if view is None else view,
                          layer_count=layers, layer_stride_bytes=stride)
        assert (e.value.variant, e.value.name) == (variant, name)

    for name in case.given:
        refused("AllocationOutOfBounds", name, **{name: kv.device_buffer(case.given[name].ptr, 8)})
        refused("DeviceMismatch", name, **{name: kv.device_buffer(1 << 20, 1 << 30)})
    refused("InvalidArgument", "alignment", kept=kv.device_buffer(case.given["kept"].ptr + 2, 1 << 10))
    refused("ZeroDimension", "layer_count", layers=0)
    refused("DimensionTooLarge", "layer_count", layers=65536)
    refused("ShapeOverflow", "", layers=3, stride=2 ** 63)
    with pytest.raises(kv.KvError) as e:  # a third layer lies behind the page
        k.keep_drafts(plan, kv.DraftBuffers(**case.given), pool.view(), layer_count=3, layer_stride_bytes=pool.layer_stride)
    assert e.value.variant == "TensorPageRegionOutOfBounds"
    view = pool.view()
    view.byte_len -= 1
    with pytest.raises(kv.KvError):
        k.keep_drafts(plan, kv.DraftBuffers(**case.given), view, **pool.call())


# ---- fork_sequences -------------------------------------------------------------------------


class Forks:
    """Sequences of `lengths` tokens over a pool: groups of them share their first full pages."""

    def __init__(self, rng, pool, lengths, groups, parents, *, append=1, spare=20, table_pages=None, prefix_held=0):
        self.pool, self.append = pool, append
        page = pool.page
        self.lengths = np.asarray(lengths, np.uint64)
        full = [n // page for n in lengths]
        self.table_pages = table_pages or max(-(-(n + append) // page) for n in lengths) + 1
        order = rng.permutation(pool.pages)
        self.tables = rng.integers(-5, 10 ** 9, (len(lengths), self.table_pages)).astype(np.int32)  # (behind the pages: anything)
        self.references = np.zeros(pool.pages, np.uint32)
        at, shared = 0, {}
        for i, n in enumerate(lengths):
            key = groups[i]
            common = min(full[j] for j in range(len(lengths)) if groups[j] == key) * 2 // 3
            if key not in shared:
                shared[key] = order[at:at + common]
                at += common
                self.references[shared[key][:prefix_held]] += 1  # as a prefix cache holds them
            own = order[at:at + -(-n // page) - common]
            at += len(own)
            row = np.concatenate([shared[key], own])
            self.tables[i, :len(row)] = row
            self.references[row] += 1
        self.free = np.full(pool.pages, -7, np.int32)
        self.free_count = spare
        self.free[:spare] = order[at:at + spare]
        self.parents = np.asarray(parents, np.uint32)
        self.result = None

    def buffers(self):
        s = len(self.parents)
        self.device = {n: hip.DeviceBuffer.from_array(a) for n, a in dict(
            parents=self.parents, lengths=self.lengths, page_tables=self.tables,
            forked_lengths=np.full(s, 77, np.uint64), forked_tables=np.full((s, self.table_pages), -77, np.int32),
            page_references=self.references, free_pages=self.free, free_count=np.asarray([self.free_count], np.uint64)).items()}
        self.plan = kv.ForkPlan.new(sequence_count=s, parent_count=len(self.lengths), table_pages=self.table_pages,
                                    page_size=self.pool.page, page_count=self.pool.pages, append_tokens=self.append)
        self.device["workspace"] = _filled(self.plan.workspace_required_bytes, 0xFF)
        return kv.ForkBuffers(**self.device)

    def run(self, k, stream=None):
        k.fork_sequences(self.plan_and_buffers()[0], self.held, self.pool.view(), stream=stream, **self.pool.call())
        hip.synchronize()
        return self.state()

    def plan_and_buffers(self):
        self.held = self.buffers()
        return self.plan, self.held

    def state(self):
        d, s = self.device, len(self.parents)
        return [d["forked_lengths"].download().view(np.uint64), d["forked_tables"].download().view(np.int32).reshape(s, -1),
                d["page_references"].download().view(np.uint32), d["free_pages"].download().view(np.int32),
                int(d["free_count"].download().view(np.uint64)[0]), self.pool.device.download()]

    def want(self):
        out = self.pool.raw.copy()

        def copy(source, to, rows):
            self.pool.move(out, int(to) * self.pool.page, self.pool.raw, int(source) * self.pool.page, rows)

        return [*ref.fork(self.parents, self.lengths, self.tables, self.references, self.free, self.free_count, self.pool.page,
                          self.append, copy), out]

    def untouched(self):
        s = len(self.parents)
        return [np.full(s, 77, np.uint64), np.full((s, self.table_pages), -77, np.int32), self.references, self.free,
                self.free_count, self.pool.raw]


def _same(got, want):
    names = ("lengths", "tables", "references", "free pages", "free count", "pool")
    for name, a, b in zip(names, got, want):
        assert np.array_equal(a, b), name


def _forks(seed, shape, lengths, groups, parents, **more):
    rng = np.random.default_rng(seed)
    pages = sum(-(-n // shape["page"]) for n in lengths) + more.get("spare", 20) + 3
    return Forks(rng, Bytes(rng, pages=pages, **shape), lengths, groups, parents, **more)


@pytest.mark.parametrize("shape", POOLS, ids=_ids)
@pytest.mark.parametrize("append", [0, 1, 70])
def test_forks(k, shape, append):
    page = shape["page"]
    # A group that goes on from one parent; one whose places change; one that ends; whole pages; one token; none.
    lengths = [3 * page + 2] * 4 + [5 * page + page // 2] * 3 + [page + 1] * 2 + [2 * page] * 2 + [1] + [0]
    groups = [0] * 4 + [1] * 3 + [2] * 2 + [3] * 2 + [4] + [5]
    parents = [2, 2, 2, 2, 6, 4, 5, NONE, NONE, 10, 10, 11, 12]
    case = _forks(21, shape, lengths, groups, parents, append=append, spare=20 + 13 * -(-append // page), prefix_held=1)
    _say(f"fork_sequences {shape} append={append}")
    got = case.run(k)
    k.check_errors()
    _same(got, case.want())


def test_more_sequences_than_before_and_fewer(k):
    shape = POOLS[0]
    case = _forks(22, shape, [100, 33], [0, 1], [0] * 9 + [1] * 5 + [NONE] * 3 + [0], spare=40)
    _same(case.run(k), case.want())
    case = _forks(23, shape, [40] * 30, [i // 3 for i in range(30)], [7, 29], spare=5)
    _same(case.run(k), case.want())
    case = _forks(24, shape, [40] * 6, [0] * 6, [NONE] * 6, spare=0)
    _same(case.run(k), case.want())
    k.check_errors()


@pytest.mark.parametrize("sequences", [1024, 1025, 3000])
def test_many_sequences(k, sequences):
    """More sequences than the plan's workgroup has threads, and more pages than it has bits."""
    rng = np.random.default_rng(25)
    pool = Bytes(rng, page=4, pages=40000, layers=1, heads=1, widths=(16,))
    lengths = rng.integers(0, 30, sequences).tolist()
    parents = rng.integers(0, sequences, sequences).astype(np.uint32)
    parents[rng.random(sequences) < 0.1] = NONE
    case = Forks(rng, pool, lengths, list(range(sequences)), parents, append=5, spare=2 * sequences + sequences)
    _same(case.run(k), case.want())
    k.check_errors()


def test_long_tables(k):
    rng = np.random.default_rng(26)
    pool = Bytes(rng, page=1, pages=9000, layers=1, heads=1, widths=(8,))
    case = Forks(rng, pool, [4000, 3000], [0, 0], [1, 1], append=3, spare=100)
    _same(case.run(k), case.want())
    k.check_errors()


@pytest.mark.parametrize("pages", [262144, 262145])
def test_many_pages(k, pages):
    """As many pages as one workgroup has bits for, and one more."""
    rng = np.random.default_rng(28)
    pool = Bytes(rng, page=2, pages=pages, layers=1, heads=1, widths=(4,))
    case = Forks(rng, pool, [801, 500, 33, 2000], [0, 0, 1, 1], [1, 1, NONE, 3], append=3, spare=100)
    _say(f"fork_sequences over {pages} pages")
    _same(case.run(k), case.want())
    k.check_errors()


def test_a_chain_of_steps(k):
    """Steps in a row without a wait, each on the tables that the one before wrote."""
    rng = np.random.default_rng(27)
    page = 8
    pool = Bytes(rng, page=page, pages=300, layers=2, heads=2, widths=(32, 32))
    case = Forks(rng, pool, [20] * 12, [i // 4 for i in range(12)], np.zeros(12), append=3, spare=150, table_pages=30)
    plan, first = case.plan_and_buffers()
    second = hip.DeviceBuffer.from_array(np.zeros(12, np.uint64)), hip.DeviceBuffer.from_array(np.zeros((12, 30), np.int32))
    d = case.device
    lengths = [d["lengths"], d["forked_lengths"], second[0]]
    tables = [d["page_tables"], d["forked_tables"], second[1]]
    state = [case.lengths, case.tables, case.references, case.free, case.free_count]
    raw = pool.raw.copy()
    held = []
    at = 0
    for step in range(12):
        parents = (rng.integers(0, 4, 12) + 4 * (np.arange(12) // 4)).astype(np.uint32)
        held.append(hip.DeviceBuffer.from_array(parents))
        to = 1 if at != 1 else 2
        k.fork_sequences(plan, kv.ForkBuffers(**{**d, "parents": held[-1], "lengths": lengths[at], "page_tables": tables[at],
                                                 "forked_lengths": lengths[to], "forked_tables": tables[to]}),
                         pool.view(), **pool.call())

        def copy(source, dest, rows):
            pool.move(raw, int(dest) * page, raw, int(source) * page, rows)

        state = list(ref.fork(parents, *state, page, 3, copy))
        at = to
    hip.synchronize()
    k.check_errors()
    got = [lengths[at].download().view(np.uint64), tables[at].download().view(np.int32).reshape(12, 30), *case.state()[2:]]
    _same(got, [*state, raw])


@pytest.mark.parametrize("what,variant", [("parent", "DeviceMetadataInvalid"), ("length", "DeviceMetadataInvalid"),
                                          ("append", "DeviceMetadataInvalid"), ("count", "DeviceMetadataInvalid"),
                                          ("free", "DevicePageIndexOutOfRange"), ("few", "DeviceOutOfPages"),
                                          ("none", "DeviceOutOfPages")])
def test_a_fork_that_does_not_hold_changes_nothing(k, what, variant):
    case = _forks(28, POOLS[0], [40, 40, 21, 16], [0, 0, 1, 2], [1, 1, 2, 3], append=4, spare=2)
    if what == "parent":
        case.parents[2] = 4
    elif what == "length":
        case.lengths[0] = 2 ** 63  # (a sequence that nothing goes on from)
    elif what == "append":
        case.append = 16 * case.table_pages - 39
    elif what == "count":
        case.free_count = case.pool.pages + 1
    elif what == "free":
        case.free[0] = case.pool.pages
    elif what == "few":
        case.free_count = 1
    elif what == "none":
        case.free_count = 0
    got = case.run(k)
    with pytest.raises(kv.KvError) as e:
        k.check_errors()
    assert e.value.variant == variant
    _same(got, case.untouched())
    k.check_errors()


def test_free_pages_to_the_last(k):
    case = _forks(29, POOLS[0], [40, 40, 21, 16], [0, 0, 1, 2], [1, 1, 2, 3], append=4, spare=2)
    _same(case.run(k), case.want())
    k.check_errors()
    # What the call does not take is not looked at.
    case = _forks(29, POOLS[0], [40, 40, 21, 16], [0, 0, 1, 2], [1, 1, 2, 3], append=4, spare=4)
    case.free[:2] = (-1, 2 ** 31 - 1)
    _same(case.run(k), case.want())
    k.check_errors()


def test_a_bad_table_entry_is_passed_on_as_none(k):
    case = _forks(30, POOLS[0], [70, 40, 21], [0, 1, 2], [0, 0, 1, 1, NONE], append=1, spare=5)
    good = case.tables.copy()
    case.tables[0, 1] = case.pool.pages
    case.tables[1, 2] = -1  # a last page, wanted twice
    got = case.run(k)
    with pytest.raises(kv.KvError) as e:
        k.check_errors()
    assert e.value.variant == "DevicePageIndexOutOfRange"
    lengths, tables = got[:2]
    assert lengths.tolist() == [70, 70, 40, 40, 0]
    assert tables[0, :5].tolist() == [good[0, 0], -1, *good[0, 2:5]] and tables[1, :4].tolist() == [good[0, 0], -1, *good[0, 2:4]]
    assert tables[2, :3].tolist() == [good[1, 0], good[1, 1], -1] and tables[3, 2] in case.free[:5]
    references = case.references.copy()
    for p in (good[0, 0], good[0, 2], good[0, 3], good[1, 0], good[1, 1]):
        references[p] += 1
    for p in (tables[1, 4], tables[3, 2]):
        references[p] += 1
    references[good[2, :2]] -= 1
    assert np.array_equal(got[2], references)
    assert got[4] == 5 - 2 + 2 and got[3][3:5].tolist() == sorted(good[2, :2])
    # The page that could be copied was; the other new one is as it was.
    raw = case.pool.raw.copy()
    case.pool.move(raw, tables[1, 4] * 16, case.pool.raw, good[0, 4] * 16, 70 % 16)
    assert np.array_equal(got[5], raw)


def test_fork_refusals(k):
    case = _forks(31, POOLS[0], [40, 40], [0, 0], [1, 1])
    plan, _ = case.plan_and_buffers()
    pool = case.pool

    def refused(variant, name, view=None, layers=pool.layers, **change):
        with pytest.raises(kv.KvError) as e:
            k.fork_sequences(plan, kv.ForkBuffers(**{**case.device, **change}), pool.view() if view is None else view,
                             layer_count=layers, layer_stride_bytes=pool.layer_stride)
        assert (e.value.variant, e.value.name) == (variant, name)

    for name, b in case.device.items():
        refused("AllocationOutOfBounds", name, **{name: kv.device_buffer(b.ptr, b.nbytes - 1)})
        refused("DeviceMismatch", name, **{name: kv.device_buffer(1 << 20, 1 << 30)})
    for a, b in (("forked_lengths", "lengths"), ("forked_tables", "page_tables"), ("forked_tables", "workspace"),
                 ("forked_lengths", "forked_tables")):
        one, two = case.device[a], case.device[b]
        big = hip.DeviceBuffer(one.nbytes + two.nbytes)
        refused("InvalidArgument", "in place", **{a: big, b: kv.device_buffer(big.ptr + one.nbytes - 16, big.nbytes - one.nbytes + 16)})
    view = pool.view()
    view.page_count -= 1
    refused("InvalidArgument", "pool", view=view)
    refused("ZeroDimension", "layer_count", layers=0)
    assert all(np.array_equal(a, b) for a, b in zip(case.state(), case.untouched()))
