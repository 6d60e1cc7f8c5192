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


def fork(parents, lengths, tables, references, free, free_count, page, append, copy):
    """The state after fork_sequences: as branch_reference.fork, but a last page that is not full goes on to a child only
    where its parent's row alone holds it."""
    before, references, free, end = references, references.copy(), free.copy(), int(free_count)
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
            if j * page >= n or (last and (p in seen or before[tables[p, j]] > 1)):
                end -= 1
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
    for number in np.flatnonzero((before > 0) & (references == 0)):
        free[end] = number
        end += 1
    return new_lengths, new_tables, references, free, end


def _want(case):
    pool, out = case.pool, case.pool.raw.copy()

    def copy(source, to, rows):
        pool.move(out, int(to) * pool.page, pool.raw, int(source) * pool.page, rows)

    return [*fork(case.parents, case.lengths, case.tables, case.references, case.free, case.free_count, pool.page, case.append,
                  copy), out]


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
