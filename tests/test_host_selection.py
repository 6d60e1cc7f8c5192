"""CPU tests of the page-selection plan (sgl_kv_page_selection_plan_new): the
sizes that it derives and what it refuses."""
import ctypes

import numpy as np
import pytest

import sgl_rocm_kv as kv


def _attention(**change):
    page, heads, dk, dv = (change.pop(n, d) for n, d in (("page", 16), ("heads", 2), ("dk", 64), ("dv", 64)))
    base = dict(query_count=3, request_count=2, sequence_slot_count=1000, slot_count=1600, query_head_count=4 * heads,
                kv_head_count=heads, query_key_head_dim=dk, value_head_dim=dv, scale=0.125, page_size=page,
                page_stride_bytes=page * heads * (dk + dv) * 2, key_in_page_offset=0,
                value_in_page_offset=page * heads * dk * 2, key_row_bytes=heads * dk * 2, value_row_bytes=heads * dv * 2)
    return kv.PagedAttentionPlan.new(**{**base, **change})


def test_sizes():
    plan = kv.PageSelectionPlan.new(_attention(), max_pages=8, first_pages=1, last_pages=2)
    assert (plan.max_pages, plan.first_pages, plan.last_pages, plan.max_sequence_length) == (8, 1, 2, 0)
    assert plan.bounds_required_bytes == 100 * 2 * 2 * 64 * 2
    assert plan.selected_required_bytes == 3 * 2 * 8 * 4
    assert plan.workspace_required_bytes > 0
    assert plan.attention.query_count == 3
    # A pool that ends inside a page has bounds for it; lists that hold every page need no scores.
    assert kv.PageSelectionPlan.new(_attention(slot_count=1601), max_pages=8).bounds_required_bytes == 101 * 512
    # Lists of every page need no scores; one page of 32 values a record of one split: none.
    assert kv.PageSelectionPlan.new(_attention(sequence_slot_count=16), max_pages=1).workspace_required_bytes == 0
    # The workspace does not grow past what the longest sequence asks for.
    short = kv.PageSelectionPlan.new(_attention(), max_pages=8, max_sequence_length=200)
    assert 0 < short.workspace_required_bytes <= plan.workspace_required_bytes


@pytest.mark.parametrize("attention,config,variant,name", [
    ({}, dict(max_pages=0), "ZeroDimension", "max_pages"),
    ({}, dict(max_pages=4, first_pages=3, last_pages=2), "InvalidArgument", "first_pages"),
    ({}, dict(max_pages=4, first_pages=2 ** 64 - 1, last_pages=2), "InvalidArgument", "first_pages"),
    ({}, dict(max_pages=4, first_pages=2, last_pages=2 ** 64 - 1), "InvalidArgument", "first_pages"),
    ({}, dict(max_pages=2 ** 31 + 1), "DimensionTooLarge", "max_pages"),
    (dict(sequence_slot_count=2 ** 36), dict(max_pages=4), "DimensionTooLarge", "sequence_pages"),
    (dict(page=2 ** 24 + 1), dict(max_pages=4), "DimensionTooLarge", "page_size"),
    (dict(dk=1025), dict(max_pages=4), "DimensionTooLarge", "query_key_head_dim"),
    (dict(dk=1024, query_head_count=160), dict(max_pages=4), "DimensionTooLarge", "query_heads_per_kv_head"),
    (dict(query_count=2 ** 27, heads=8), dict(max_pages=4), "DimensionTooLarge", "workgroups"),
    (dict(query_count=2 ** 32 - 1, heads=2 ** 20, query_head_count=2 ** 20), dict(max_pages=4), "DimensionTooLarge",
     "workgroups"),
])
def test_refusals(attention, config, variant, name):
    with pytest.raises(kv.KvError) as e:
        kv.PageSelectionPlan.new(_attention(**attention), **config)
    assert (e.value.variant, e.value.name) == (variant, name)


def test_an_edited_attention_plan_is_checked_again():
    plan = _attention()
    plan._c.config.query_head_count = 7
    with pytest.raises(kv.KvError) as e:
        kv.PageSelectionPlan.new(plan, max_pages=4)
    assert e.value.variant == "QueryHeadsNotDivisibleByKvHeads"


def test_null_arguments():
    plan = kv.PageSelectionPlan.new(_attention(), max_pages=8)
    buffers = kv.PageSelectionBuffers()
    lib = kv.lib()
    for rc in (lib.sgl_kv_page_selection_plan_new(None, None, None),
               lib.sgl_rocm_kv_select_pages(None, ctypes.byref(plan._c), ctypes.byref(buffers._c), None),
               lib.sgl_rocm_kv_selected_attention(None, ctypes.byref(plan._c), ctypes.byref(buffers._c), None),
               lib.sgl_rocm_kv_page_bounds(None, None, None, None, 1, None, None)):
        assert kv.status_name(rc) == "InvalidArgument"


def test_unknown_buffers_are_refused():
    with pytest.raises(TypeError):
        kv.PageSelectionBuffers(pages=kv.device_buffer(0, 0))


def test_random_plans_never_overflow():
    """Sizes over the whole range of 64 bits: a plan, or a named refusal."""
    rng = np.random.default_rng(1)
    for _ in range(3000):
        def size(most):
            return int(2 ** rng.uniform(0, most))
        heads, dk, dv, page = size(8), size(11), size(11), size(26)
        try:
            a = _attention(page=page, heads=heads, dk=dk, dv=dv, query_count=size(33), query_head_count=heads * size(9),
                           sequence_slot_count=size(60), slot_count=size(40))
            p = kv.PageSelectionPlan.new(a, max_pages=size(33), max_sequence_length=size(60))
        except kv.KvError as e:
            assert e.variant in ("DimensionTooLarge", "ShapeOverflow"), e
            continue
        assert p.selected_required_bytes == a.query_count * heads * p.max_pages * 4
