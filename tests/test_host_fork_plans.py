"""CPU tests of the plan of forks that keep reserved pages."""
import pytest

import sgl_rocm_kv as kv

FORKS = dict(sequence_count=5, parent_count=3, table_pages=7, page_size=16, page_count=100)


def test_keep_reserved():
    plain, keeps = kv.ForkPlan.new(**FORKS), kv.ForkPlan.new(**FORKS, keep_reserved=True)
    assert (plain.keep_reserved, keeps.keep_reserved) == (0, 1)
    assert keeps.workspace_required_bytes >= plain.workspace_required_bytes + 4 * FORKS["parent_count"]
    assert keeps.forked_tables_required_bytes == plain.forked_tables_required_bytes


@pytest.mark.parametrize("change,variant,name", [
    (dict(keep_reserved=2), "InvalidArgument", "keep_reserved"),
    (dict(keep_reserved=True, table_pages=2 ** 20 + 1), "DimensionTooLarge", "table_pages"),
])
def test_refusals(change, variant, name):
    with pytest.raises(kv.KvError) as e:
        kv.ForkPlan.new(**{**FORKS, **change})
    assert (e.value.variant, e.value.name) == (variant, name)
    kv.ForkPlan.new(**{**FORKS, "table_pages": 2 ** 20, "keep_reserved": True})
    kv.ForkPlan.new(**{**FORKS, "table_pages": 2 ** 20 + 1})
