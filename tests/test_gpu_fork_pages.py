"""GPU tests of which pages fork_sequences shares, copies and keeps, against a restatement of its own that goes sequence
by sequence. Tables, counts, lists and pages are compared exactly."""
import numpy as np
import pytest

import sgl_rocm_kv as kv
from branch_reference import NONE
from sgl_rocm_kv import hip
from test_gpu_branches import POOLS, Bytes, Forks, _ids, _same
from test_gpu_selection import _say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def k():
    if hip.device_count() == 0:
        pytest.fail("no GPU visible: the gpu tests need an MI355X")
    ctx = kv.RocmKvPairCopyKernels(0)
    yield ctx
    ctx.close()


def _pages(n, table, page, keep):
    """Entries of a row of n tokens that are pages of it."""
    end = -(-int(n) // page)
    while keep and end < len(table) and table[end] >= 0:
        end += 1
    return end


def fork(parents, lengths, tables, references, free, free_count, page, append, copy, keep=False):
    """The state after fork_sequences: as branch_reference.fork, but a last page that is not full goes on to a child only
    where its parent's row alone holds it; with `keep`, pages behind a row's own go on with its lowest child."""
    before, references, free, end = references, references.copy(), free.copy(), int(free_count)
    new_lengths = np.zeros(len(parents), np.uint64)
    new_tables = np.full((len(parents), tables.shape[1]), -1, np.int32)
    seen = set()
    for s, p in enumerate(parents):
        if p == NONE:
            continue
        n = int(lengths[p])
        new_lengths[s] = n
        held = _pages(n, tables[p], page, keep and p not in seen)
        for j in range(max(held, -(-(n + append) // page))):
            last = j == n // page and n % page > 0
            if j >= held or (last and (p in seen or before[tables[p, j]] > 1)):
                end -= 1
                new_tables[s, j] = free[end]
                if last:
                    copy(tables[p, j], free[end], n % page)
            else:
                new_tables[s, j] = tables[p, j]
            references[new_tables[s, j]] += 1
        seen.add(p)
    for n, table in zip(lengths, tables):
        for j in range(_pages(n, table, page, keep)):
            references[table[j]] -= 1
    for number in np.flatnonzero((before > 0) & (references == 0)):
        free[end] = number
        end += 1
    return new_lengths, new_tables, references, free, end


def _want(case, keep=False):
    pool, out = case.pool, case.pool.raw.copy()

    def copy(source, to, rows):
        pool.move(out, int(to) * pool.page, pool.raw, int(source) * pool.page, rows)

    return [*fork(case.parents, case.lengths, case.tables, case.references, case.free, case.free_count, pool.page, case.append,
                  copy, keep), out]


WAYS = [None, 9000]  # entries of a table's row: as few as there are, and more than one workgroup takes


@pytest.mark.parametrize("table_pages", WAYS)
@pytest.mark.parametrize("shape", POOLS[:5], ids=_ids)
def test_a_last_page_that_more_than_its_parent_holds(k, shape, table_pages):
    """Two sequences on the same partial page, one that the caller holds, a shorter sequence inside another's full page:
    no child goes on writing to any of these."""
    page = shape["page"]
    half = page // 2 + 1
    lengths = [2 * page + half] * 2 + [page + half] * 2 + [3 * page, page + half, 2 * page + 1] + [half] * 2
    #          0, 1: one page      2: held by the caller   4, 5: 5 ends inside 4's   6: alone    7, 8: one page, 8 ends
    parents = [0, 0, 1, 2, 3, 3, 4, 5, 5, 6, 6, 7, NONE]
    rng = np.random.default_rng(61)
    pool = Bytes(rng, pages=40, **shape)
    case = Forks(rng, pool, lengths, list(range(len(lengths))), parents, append=1, spare=20, table_pages=table_pages)

    def same(a, b, entries):
        for j in entries:
            case.references[case.tables[b, j]] = 0
            case.tables[b, j] = case.tables[a, j]
            case.references[case.tables[a, j]] += 1

    same(0, 1, range(3))
    case.references[case.tables[2, 1]] += 1
    same(4, 5, range(2))
    same(7, 8, range(1))
    _say(f"fork_sequences, shared last pages, {shape} {table_pages}")
    got, want = case.run(k), _want(case)
    k.check_errors()
    _same(got, want)
    tables, references = got[1], got[2]
    held = case.tables[2, 1]
    assert references[held] == 1  # the caller's
    writable = [tables[s, int(n) // page] for s, n in enumerate(got[0]) if parents[s] != NONE]
    assert len(set(writable)) == len(writable) and all(references[p] == 1 for p in writable)


@pytest.mark.parametrize("table_pages", WAYS)
def test_a_step_after_a_shared_one(k, table_pages):
    """A second step on what the first wrote: every page of it is its sequence's own, so that lowest children take them over."""
    rng = np.random.default_rng(62)
    pool = Bytes(rng, pages=60, **POOLS[0])
    case = Forks(rng, pool, [40, 40, 25], [0, 1, 2], [0, 1, 1, 2], append=1, spare=30, table_pages=table_pages)
    for j in range(3):
        case.references[case.tables[1, j]] = 0
        case.tables[1, j] = case.tables[0, j]
        case.references[case.tables[0, j]] += 1
    got, want = case.run(k), _want(case)
    _same(got, want)
    second = Forks.__new__(Forks)
    second.__dict__.update(pool=pool, append=1, table_pages=case.table_pages, lengths=want[0], tables=want[1], references=want[2],
                           free=want[3], free_count=want[4], parents=np.asarray([3, 1, 1, 0], np.uint32))
    pool.raw = want[5]
    got, want = second.run(k), _want(second)
    k.check_errors()
    _same(got, want)
    assert got[1][0, 1] == second.tables[3, 1] and got[1][1, 2] == second.tables[1, 2]


class Reserved(Forks):
    """Forks whose old rows hold `reserved` pages behind their own, and -1 behind these."""

    def __init__(self, rng, pool, lengths, groups, parents, *, reserved, **more):
        super().__init__(rng, pool, lengths, groups, parents, **more)
        for n, extra, row in zip(lengths, reserved, self.tables):
            end = -(-n // pool.page)
            row[end:] = -1
            for j in range(end, end + extra):
                self.free_count -= 1
                row[j] = self.free[self.free_count]
                self.references[row[j]] = 1

    def buffers(self):
        super().buffers()
        self.plan = kv.ForkPlan.new(sequence_count=len(self.parents), parent_count=len(self.lengths), page_size=self.pool.page,
                                    table_pages=self.table_pages, page_count=self.pool.pages, append_tokens=self.append,
                                    keep_reserved=True)
        self.device["workspace"] = hip.DeviceBuffer.from_array(np.full(self.plan.workspace_required_bytes, 0xFF, np.uint8))
        return kv.ForkBuffers(**self.device)


@pytest.mark.parametrize("table_pages", WAYS)
@pytest.mark.parametrize("append", [0, 1, 40])
@pytest.mark.parametrize("shape", POOLS[:5], ids=_ids)
def test_reserved_pages(k, shape, append, table_pages):
    """Kept by the lowest child, taken before new ones, freed where there is no child; more than are wanted, too, and of a
    sequence without tokens; beside a last page that the caller holds, and a row that is full to its end."""
    page = shape["page"]
    half = page // 2
    #          one child, two, none, whole pages, no tokens, shared last page, none of both
    lengths = [2 * page + half, page + half, page + 1, 3 * page, 0, 2 * page + half, 4 * page, page + half]
    reserved = [1, 2, 3, 1, 2, 2, 9, 0]
    parents = [1, 0, 1, 3, 3, 4, 5, 5, 6, 7, NONE]
    rng = np.random.default_rng(63)
    pool = Bytes(rng, pages=90 + 11 * -(-append // page), **shape)
    case = Reserved(rng, pool, lengths, list(range(8)), parents, reserved=reserved, append=append,
                    spare=50 + 11 * -(-append // page), table_pages=table_pages or max(13, 5 + -(-append // page)))
    case.references[case.tables[5, 2]] += 1
    _say(f"fork_sequences, reserved pages, {shape} append={append} {case.table_pages}")
    got, want = case.run(k), _want(case, True)
    k.check_errors()
    _same(got, want)


def _owned(tables, lengths, page):
    """Every page of the rows, once."""
    return np.unique(np.concatenate([row[:_pages(n, row, page, True)] for n, row in zip(lengths, tables)]))


@pytest.mark.parametrize("table_pages", [40, 9000])
def test_no_page_is_lost_over_steps(k, table_pages):
    """Steps that reserve more than the sequences grow into: after each one every page is free or held by a row, and the
    second way to see it, the counts, agree."""
    rng = np.random.default_rng(64)
    page, sequences = 8, 12
    pool = Bytes(rng, page=page, pages=160, layers=2, heads=2, widths=(32, 32))
    case = Reserved(rng, pool, [20, 24, 16, 1, 8, 9, 20, 31, 0, 7, 15, 33], list(range(sequences)), range(sequences),
                    reserved=[0] * sequences, append=20, spare=120, table_pages=table_pages)
    total = len(_owned(case.tables, case.lengths, page)) + case.free_count
    kept = 0
    for step in range(20):
        got, want = case.run(k), _want(case, True)
        k.check_errors()
        _same(got, want)
        lengths, tables, references, free, free_count, raw = want
        owned = _owned(tables, lengths, page)
        assert len(owned) + free_count == total and not np.intersect1d(owned, free[:free_count]).size, step
        assert np.array_equal(np.flatnonzero(references), owned)
        kept += int(sum((row >= 0).sum() for row in tables) > sum(-(-int(n) // page) for n in lengths))
        # The next step: each sequence has written some of what it could, and a few take others' places.
        lengths = lengths + rng.integers(0, 3, sequences).astype(np.uint64) * (rng.random(sequences) < 0.7)
        parents = np.arange(sequences)
        moved = rng.random(sequences) < 0.3
        parents[moved] = rng.integers(0, sequences, moved.sum())
        pool.raw = raw
        case.lengths, case.tables, case.references, case.free, case.free_count = lengths.astype(np.uint64), tables, references, free, free_count
        case.parents = parents.astype(np.uint32)
    assert kept == 20


@pytest.mark.parametrize("table_pages", WAYS)
def test_what_ends_reserved_pages(k, table_pages):
    """An entry outside the pool ends them and is reported; what is behind it is not looked at."""
    rng = np.random.default_rng(65)
    pool = Bytes(rng, pages=40, **POOLS[0])
    case = Reserved(rng, pool, [20, 33], [0, 1], [0, 1, 1], reserved=[2, 1], append=1, spare=12, table_pages=table_pages or 9)
    case.tables[0, 3] = 40  # the second of two
    case.tables[1, 5] = -7  # behind a -1
    got = case.run(k)
    with pytest.raises(kv.KvError) as e:
        k.check_errors()
    assert e.value.variant == "DevicePageIndexOutOfRange"
    assert got[1][0, :5].tolist() == [*case.tables[0, :3], -1, -1] and got[1][1, 3] == case.tables[1, 3] and got[1][1, 4] == -1
    case.tables[0, 3] = -1
    got, want = case.run(k), _want(case, True)
    k.check_errors()
    _same(got, want)


def test_without_them_what_is_behind_is_not_looked_at(k):
    """The default: entries behind a sequence's pages may be anything."""
    rng = np.random.default_rng(66)
    pool = Bytes(rng, pages=40, **POOLS[0])
    case = Forks(rng, pool, [20, 33], [0, 1], [0, 1, 1], append=17, spare=12)
    assert (case.tables[0, 2:] != -1).all()
    got, want = case.run(k), _want(case)
    k.check_errors()
    _same(got, want)
