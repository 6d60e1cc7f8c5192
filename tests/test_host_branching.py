"""CPU tests of the plans of tree_attention, keep_drafts, select_beams and
fork_sequences: the sizes that they derive and what they refuse."""
import ctypes

import numpy as np
import pytest

import sgl_rocm_kv as kv
from test_host_selection import _attention

DRAFTS = dict(request_count=3, sequence_slot_count=100, max_kept=8)
BEAMS = dict(request_count=3, beam_count=4, vocab_size=1000, max_kept=5)
FORKS = dict(sequence_count=5, parent_count=3, table_pages=7, page_size=16, page_count=100)


def _tree(attention=None, **config):
    return kv.TreeAttentionPlan.new(_attention(**(attention or {})), **{**dict(mask_words=1), **config})


def test_sizes():
    tree = _tree(mask_words=3)
    assert (tree.mask_words, tree.max_sequence_length, tree.masks_required_bytes) == (3, 0, 3 * 3 * 8)
    assert tree.attention.query_count == 3 and tree.workspace_required_bytes > 0
    drafts = kv.DraftPlan.new(**DRAFTS)
    assert (drafts.request_lengths_required_bytes, drafts.request_slot_offsets_required_bytes) == (24, 32)
    assert (drafts.sequence_slots_required_bytes, drafts.kept_required_bytes) == (800, 3 * 8 * 4)
    beams = kv.BeamPlan.new(**BEAMS)
    assert (beams.logits_required_bytes, beams.scores_required_bytes) == (12 * 1000 * 2, 48)
    assert beams.best_scores_required_bytes == beams.best_parents_required_bytes == beams.best_tokens_required_bytes == 60
    assert beams.workspace_required_bytes > 0
    # The last row ends with its last logit.
    assert kv.BeamPlan.new(**BEAMS, dtype="f32", row_stride=1024).logits_required_bytes == (11 * 1024 + 1000) * 4
    forks = kv.ForkPlan.new(**FORKS, append_tokens=9)
    assert (forks.parents_required_bytes, forks.lengths_required_bytes, forks.forked_lengths_required_bytes) == (20, 24, 40)
    assert (forks.page_tables_required_bytes, forks.forked_tables_required_bytes) == (3 * 7 * 4, 5 * 7 * 4)
    assert (forks.page_references_required_bytes, forks.free_pages_required_bytes, forks.free_count_required_bytes) == (400, 400, 8)
    assert forks.append_tokens == 9 and forks.workspace_required_bytes > 0


@pytest.mark.parametrize("dk", [64, 128, 256, 40])
@pytest.mark.parametrize("requests,queries,slots", [(1, 1, 1), (1, 16, 2064), (32, 544, 140000), (64, 64, 10 ** 7),
                                                    (65, 1000, 200000), (4, 4096, 9000), (4, 4097, 9000), (1000, 9000, 10 ** 8)])
def test_the_tree_workspace_stays_in_bounds(dk, requests, queries, slots):
    """A query head's records: at most a few for each workgroup that its request can have, whatever the longest sequence."""
    plan = _tree(dict(dk=dk, dv=dk, request_count=requests, query_count=queries, sequence_slot_count=slots))
    heads = plan.attention.query_head_count
    records = plan.workspace_required_bytes / (queries * heads * 4 * (dk + 32))
    assert records <= max(8, 2 * 2048 / requests + 3)
    # It does not grow past what the longest sequence asks for.
    short = _tree(dict(dk=dk, dv=dk, request_count=requests, query_count=queries, sequence_slot_count=slots),
                  max_sequence_length=min(slots, 64))
    assert short.workspace_required_bytes <= max(64, plan.workspace_required_bytes)


@pytest.mark.parametrize("attention,config,variant,name", [
    ({}, dict(mask_words=0), "ZeroDimension", "mask_words"),
    ({}, dict(mask_words=17), "DimensionTooLarge", "mask_words"),
    ({}, dict(mask_words=2 ** 64 - 1), "DimensionTooLarge", "mask_words"),
    (dict(sequence_slot_count=2 ** 36), {}, "DimensionTooLarge", "max_sequence_length"),
    (dict(dk=1025), {}, "DimensionTooLarge", "query_key_head_dim"),
    (dict(query_count=2 ** 27, heads=8), {}, "DimensionTooLarge", "workgroups"),
    (dict(query_count=2 ** 32 - 1, heads=2 ** 20, query_head_count=2 ** 20), {}, "DimensionTooLarge", "workgroups"),
])
def test_tree_refusals(attention, config, variant, name):
    with pytest.raises(kv.KvError) as e:
        _tree(attention, **config)
    assert (e.value.variant, e.value.name) == (variant, name)


@pytest.mark.parametrize("plan,base,change,variant,name", [
    *((kv.DraftPlan, DRAFTS, {n: 0}, "ZeroDimension", n) for n in DRAFTS),
    (kv.DraftPlan, DRAFTS, dict(max_kept=2 ** 31 + 1), "DimensionTooLarge", "max_kept"),
    (kv.DraftPlan, DRAFTS, dict(request_count=2 ** 64 - 1), "ShapeOverflow", None),
    (kv.DraftPlan, DRAFTS, dict(request_count=2 ** 61), "ShapeOverflow", None),
    (kv.DraftPlan, DRAFTS, dict(sequence_slot_count=2 ** 61), "ShapeOverflow", None),
    *((kv.BeamPlan, BEAMS, {n: 0}, "ZeroDimension", n) for n in BEAMS),
    (kv.BeamPlan, BEAMS, dict(row_stride=999), "InvalidArgument", "row_stride"),
    (kv.BeamPlan, BEAMS, dict(dtype="fp8_e4m3"), "InvalidArgument", "dtype"),
    (kv.BeamPlan, BEAMS, dict(max_kept=129), "DimensionTooLarge", "max_kept"),
    (kv.BeamPlan, BEAMS, dict(beam_count=2 ** 20), "DimensionTooLarge", "beam_count"),
    (kv.BeamPlan, BEAMS, dict(vocab_size=2 ** 40), "DimensionTooLarge", "vocab_size"),
    (kv.BeamPlan, BEAMS, dict(request_count=2 ** 32), "DimensionTooLarge", "request_count"),
    (kv.BeamPlan, BEAMS, dict(request_count=2 ** 32 - 1), "DimensionTooLarge", "workgroups"),
    (kv.BeamPlan, BEAMS, dict(request_count=2 ** 23, beam_count=1), "DimensionTooLarge", "workgroups"),
    (kv.BeamPlan, BEAMS, dict(row_stride=2 ** 63), "ShapeOverflow", None),
    *((kv.ForkPlan, FORKS, {n: 0}, "ZeroDimension", n) for n in FORKS),
    (kv.ForkPlan, FORKS, dict(append_tokens=2 ** 32), "DimensionTooLarge", "append_tokens"),
    (kv.ForkPlan, FORKS, dict(page_count=2 ** 31), "DimensionTooLarge", "page_count"),
    (kv.ForkPlan, FORKS, dict(table_pages=2 ** 32), "DimensionTooLarge", "table_pages"),
    (kv.ForkPlan, FORKS, dict(sequence_count=2 ** 64 - 1), "DimensionTooLarge", "sequence_count"),
    (kv.ForkPlan, FORKS, dict(sequence_count=2 ** 24, parent_count=2 ** 24), "DimensionTooLarge", "workgroups"),
])
def test_refusals(plan, base, change, variant, name):
    with pytest.raises(kv.KvError) as e:
        plan.new(**{**base, **change})
    assert e.value.variant == variant and (name is None or e.value.name == name)


def test_an_edited_attention_plan_is_checked_again():
    plan = _attention()
    plan._c.config.query_head_count = 7
    with pytest.raises(kv.KvError) as e:
        kv.TreeAttentionPlan.new(plan, mask_words=1)
    assert e.value.variant == "QueryHeadsNotDivisibleByKvHeads"


def test_null_arguments():
    lib = kv.lib()
    for rc in (lib.sgl_kv_tree_attention_plan_new(None, None, None), lib.sgl_kv_draft_plan_new(None, None),
               lib.sgl_kv_beam_plan_new(None, None), lib.sgl_kv_fork_plan_new(None, None),
               lib.sgl_rocm_kv_tree_attention(None, ctypes.byref(_tree()._c), ctypes.byref(kv.TreeAttentionBuffers()._c), None),
               lib.sgl_rocm_kv_keep_drafts(None, ctypes.byref(kv.DraftPlan.new(**DRAFTS)._c),
                                           ctypes.byref(kv.DraftBuffers()._c), None, 1, 0, None),
               lib.sgl_rocm_kv_select_beams(None, ctypes.byref(kv.BeamPlan.new(**BEAMS)._c),
                                            ctypes.byref(kv.BeamBuffers()._c), None),
               lib.sgl_rocm_kv_fork_sequences(None, ctypes.byref(kv.ForkPlan.new(**FORKS)._c),
                                              ctypes.byref(kv.ForkBuffers()._c), None, 1, 0, None)):
        assert kv.status_name(rc) == "InvalidArgument"


@pytest.mark.parametrize("buffers", [kv.TreeAttentionBuffers, kv.DraftBuffers, kv.BeamBuffers, kv.ForkBuffers])
def test_unknown_buffers_are_refused(buffers):
    with pytest.raises(TypeError):
        buffers(pages=kv.device_buffer(0, 0))


def test_random_plans_never_overflow():
    """Sizes over the whole range of 64 bits: a plan whose sizes hold, or a named refusal."""
    rng = np.random.default_rng(1)

    def size(most):
        return int(2 ** rng.uniform(0, most))

    made = dict.fromkeys("tdbf", 0)
    for _ in range(2000):
        heads = size(8)
        cases = [
            ("t", lambda: _tree(dict(page=size(26), heads=heads, dk=size(11), dv=size(11), query_count=size(33),
                                     query_head_count=heads * size(9), request_count=size(30), sequence_slot_count=size(60),
                                     slot_count=size(40)), mask_words=size(5), max_sequence_length=size(60))),
            ("d", lambda: kv.DraftPlan.new(request_count=size(62), sequence_slot_count=size(62), max_kept=size(33))),
            ("b", lambda: kv.BeamPlan.new(request_count=size(33), beam_count=size(10), vocab_size=size(40), max_kept=size(8),
                                          row_stride=size(62) if rng.random() < 0.5 else 0)),
            ("f", lambda: kv.ForkPlan.new(sequence_count=size(26), parent_count=size(26), table_pages=size(33),
                                          page_size=size(33), page_count=size(33), append_tokens=size(33)))]
        for name, make in cases:
            try:
                p = make()
            except kv.KvError as e:
                assert e.variant in ("DimensionTooLarge", "ShapeOverflow") or e.name == "row_stride", e
                continue
            made[name] += 1
            if name == "t":
                assert p.masks_required_bytes == p.attention.query_count * p.mask_words * 8
            elif name == "d":
                assert p.kept_required_bytes == p.request_count * p.max_kept * 4
            elif name == "b":
                rows, stride = p.request_count * p.beam_count, p.row_stride or p.vocab_size
                assert p.logits_required_bytes == ((rows - 1) * stride + p.vocab_size) * 2
                assert p.workspace_required_bytes >= 8 * rows * p.max_kept
            else:
                assert p.page_tables_required_bytes == p.parent_count * p.table_pages * 4
                assert p.workspace_required_bytes >= 4 * (2 * p.parent_count + p.sequence_count)
    assert min(made.values()) > 50, made
