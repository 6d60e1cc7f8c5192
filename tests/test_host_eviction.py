"""CPU tests of the eviction plans (sgl_kv_weight_plan_new,
sgl_kv_eviction_plan_new): the sizes that they derive and what they refuse."""
import ctypes

import numpy as np
import pytest

import sgl_rocm_kv as kv
from test_host_selection import _attention


def test_weight_plan_sizes():
    plan = kv.WeightAccumulationPlan.new(_attention())
    assert plan.weights_required_bytes == 2 * 1000 * 4
    assert plan.workspace_required_bytes >= 3 * 8 * 8 and plan.attention.request_count == 2
    short = kv.WeightAccumulationPlan.new(_attention(), max_sequence_length=100)
    assert short.max_sequence_length == 100 and 0 < short.workspace_required_bytes <= plan.workspace_required_bytes


@pytest.mark.parametrize("change,name", [
    (dict(dk=1025), "query_key_head_dim"), (dict(query_count=2 ** 27, heads=8), "workgroups"),
    (dict(request_count=2 ** 30), "workgroups"), (dict(sequence_slot_count=2 ** 40), "workgroups")])
def test_weight_plan_refusals(change, name):
    with pytest.raises(kv.KvError) as e:
        kv.WeightAccumulationPlan.new(_attention(**change))
    assert (e.value.variant, e.value.name) == ("DimensionTooLarge", name)


def _plan(**change):
    return kv.EvictionPlan.new(**{**dict(request_count=3, kv_head_count=2, sequence_slot_count=1000, max_kept=40,
                                         destination_slot_count=120), **change})


def test_eviction_plan_sizes():
    p = _plan(first_tokens=4, last_tokens=16)
    assert (p.max_kept, p.first_tokens, p.last_tokens, p.destination_slot_count) == (40, 4, 16, 120)
    assert p.kept_required_bytes == 3 * 2 * 40 * 4 and p.weights_required_bytes == 2 * 1000 * 4
    assert p.request_lengths_required_bytes == 24 and p.request_slot_offsets_required_bytes == 32
    assert p.sequence_slots_required_bytes == 8000 and p.destination_slots_required_bytes == 960
    assert p.destination_weights_required_bytes == 2 * 120 * 4


def test_the_eviction_plans_workspace_is_reserved():
    for change in ({}, dict(sequence_slot_count=2 ** 31), dict(request_count=2 ** 20, max_kept=2 ** 20)):
        assert _plan(**change).workspace_required_bytes == 0


@pytest.mark.parametrize("change,variant,name", [
    *[({n: 0}, "ZeroDimension", n) for n in ("request_count", "kv_head_count", "sequence_slot_count", "max_kept")],
    (dict(first_tokens=30, last_tokens=11), "InvalidArgument", "first_tokens"),
    (dict(first_tokens=2 ** 64 - 1, last_tokens=2), "InvalidArgument", "first_tokens"),
    (dict(last_tokens=2 ** 64 - 1), "InvalidArgument", "first_tokens"),
    (dict(max_kept=2 ** 31 + 1), "DimensionTooLarge", "max_kept"),
    (dict(sequence_slot_count=2 ** 32), "DimensionTooLarge", "max_sequence_length"),
    (dict(request_count=2 ** 22), "DimensionTooLarge", "workgroups"),
    (dict(request_count=2 ** 60), "ShapeOverflow", ""),
])
def test_eviction_plan_refusals(change, variant, name):
    with pytest.raises(kv.KvError) as e:
        _plan(**change)
    assert (e.value.variant, e.value.name) == (variant, name)


def test_a_long_slot_list_of_short_requests_is_taken():
    assert _plan(sequence_slot_count=2 ** 33, max_sequence_length=1000).max_sequence_length == 1000


def test_null_arguments():
    plan, weights = _plan(), kv.WeightAccumulationPlan.new(_attention())
    lib, b, wb = kv.lib(), kv.EvictionBuffers(), kv.WeightAccumulationBuffers()
    for rc in (lib.sgl_kv_weight_plan_new(None, 0, None), lib.sgl_kv_eviction_plan_new(None, None),
               lib.sgl_rocm_kv_accumulate_weights(None, ctypes.byref(weights._c), ctypes.byref(wb._c), None),
               lib.sgl_rocm_kv_select_tokens(None, ctypes.byref(plan._c), ctypes.byref(b._c), None),
               lib.sgl_rocm_kv_compact_tokens(None, ctypes.byref(plan._c), ctypes.byref(b._c), None, None, None)):
        assert kv.status_name(rc) == "InvalidArgument"
    for cls in (kv.EvictionBuffers, kv.WeightAccumulationBuffers):
        with pytest.raises(TypeError):
            cls(values=kv.device_buffer(0, 0))


def test_random_plans_never_overflow():
    rng = np.random.default_rng(1)

    def size(most):
        return int(2 ** rng.uniform(0, most))
    for _ in range(3000):
        try:
            p = kv.EvictionPlan.new(request_count=size(40), kv_head_count=size(40), sequence_slot_count=size(63),
                                    max_kept=size(33), destination_slot_count=size(63), max_sequence_length=size(63))
            assert p.kept_required_bytes == p.request_count * p.kv_head_count * p.max_kept * 4
        except kv.KvError as e:
            assert e.variant in ("DimensionTooLarge", "ShapeOverflow"), e


def test_random_weight_plans_never_overflow():
    rng = np.random.default_rng(2)

    def size(most):
        return int(2 ** rng.uniform(0, most))
    for _ in range(3000):
        heads = size(8)
        try:
            a = _attention(page=size(20), heads=heads, dk=int(rng.choice([64, 128, 256, size(11)])), query_count=size(33),
                           query_head_count=heads * size(9), request_count=size(33), sequence_slot_count=size(60))
            p = kv.WeightAccumulationPlan.new(a, max_sequence_length=size(60))
            assert p.workspace_required_bytes >= a.query_count * a.query_head_count * 8
        except kv.KvError as e:
            assert e.variant in ("DimensionTooLarge", "ShapeOverflow"), e
