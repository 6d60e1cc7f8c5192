"""GPU tests of select_beams where a workgroup takes several rounds of a row: large batches, which are made of a few
requests over and over, so that the 64-bit restatement in branch_reference.py has few rows to sort.

Scores: test_gpu_beams.py's bound, 2^-17 for a sum and half a step of fp32 of the score, holds for one round, of 32
roundings a thread. A further round adds one rounding of the thread's total, in 64 bits, and where its maximum grows a
factor exp2(y), off by 2^-23 of itself and by 2^-23 |y| from y's own roundings; the y of the exponentials that count
add up to less than 22. So 2^-17 + 2^-18 + rounds 2^-23, and 2^-17 where no maximum grows."""
import numpy as np
import pytest

import sgl_rocm_kv as kv
from branch_reference import NONE, best_beams
from selection_reference import bf16, f64
from sgl_rocm_kv import hip
from test_gpu_selection import _filled, _say

pytestmark = pytest.mark.gpu

CHUNK, WORKGROUPS = 8192, 2048  # logits of a round, and the workgroups up to which each takes one


@pytest.fixture(scope="module")
def k():
    if hip.device_count() == 0:
        pytest.fail("no GPU visible: the gpu tests need an MI355X")
    ctx = kv.RocmKvPairCopyKernels(0)
    yield ctx
    ctx.close()


def _rounds(rows, vocab):
    chunks = -(-vocab // CHUNK)
    return max(1, min(chunks, rows * chunks // WORKGROUPS))


def _select(k, raw, scores, times, keep, dtype, pad=0, shift=0):
    """[times][request][keep] of each output for the requests raw[request][beam][vocab], taken `times` times over."""
    requests, beams, vocab = raw.shape
    stride = vocab + pad
    one = np.full((requests * beams, stride), 0x7FC0 if dtype == "bf16" else np.nan, raw.dtype)
    one[:, :vocab] = raw.reshape(-1, vocab)
    flat = np.concatenate([np.zeros(shift, raw.dtype), np.tile(one.reshape(-1), times)])
    flat = flat[:len(flat) - pad] if pad else flat  # the last row has nothing behind it
    plan = kv.BeamPlan.new(request_count=requests * times, beam_count=beams, vocab_size=vocab, max_kept=keep, dtype=dtype,
                           row_stride=stride if pad else 0)
    out = {n: _filled(4 * requests * times * keep) for n in ("best_scores", "best_parents", "best_tokens")}
    k.select_beams(plan, kv.BeamBuffers(
        logits=hip.DeviceBuffer.from_array(flat), logits_offset=shift * raw.itemsize,
        scores=hip.DeviceBuffer.from_array(np.tile(scores, (times, 1)).astype(np.float32)),
        workspace=_filled(plan.workspace_required_bytes, 0xFF), **out))
    hip.synchronize()
    k.check_errors()
    return [out[n].download().view(t).reshape(times, requests, keep)
            for n, t in (("best_scores", np.float32), ("best_parents", np.uint32), ("best_tokens", np.uint32))]


def _check(k, logits, scores, times, keep, dtype, rounds, pad=0, shift=0):
    raw = bf16(logits) if dtype == "bf16" else np.asarray(logits, np.float32)
    requests, beams, vocab = raw.shape
    assert _rounds(requests * times * beams, vocab) == rounds
    _say(f"select_beams {requests * times}x{beams}x{vocab} keep={keep} {dtype} pad={pad} shift={shift}: {rounds} rounds")
    scores = np.asarray(scores, np.float32)
    got = _select(k, raw, scores, times, keep, dtype, pad, shift)
    exact = f64(raw) if dtype == "bf16" else raw.astype(np.float64)
    want, parents, tokens = best_beams(exact, scores.astype(np.float64), keep)
    has = parents != NONE
    first = (requests * beams * np.arange(times, dtype=np.uint32))[:, None, None]
    assert np.array_equal(got[2], np.broadcast_to(tokens, got[2].shape))
    assert np.array_equal(got[1], np.where(has, parents + first, NONE))
    assert (got[0][:, ~has] == -np.inf).all()
    error = np.abs(got[0][:, has] - want[has])
    bound = 2.0 ** -17 + 2.0 ** -18 + rounds * 2.0 ** -23 + 2.0 ** -24 * np.abs(want[has])
    if has.any():
        _say(f"beams: largest error {error.max():.3g}, {(error / bound).max():.3f} of the bound")
    assert (error <= bound).all()
    return got


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab,rows,rounds,keep,pad,shift", [
    (60000, 512, 2, 8, 0, 0),     # eight chunks in four splits of two
    (40000, 1024, 2, 8, 1, 0),    # five: the last split has one
    (50257, 1024, 3, 10, 47, 3),  # seven: the last has one of three, odd rows
    (17000, 2048, 3, 5, 3, 1),    # all three in one split
    (20001, 1024, 1, 4, 0, 1),    # one round a split, for comparison
    (33000, 2048, 5, 100, 0, 0),  # all of five, and more kept than a wave has lanes
])
def test_rounds(k, dtype, vocab, rows, rounds, keep, pad, shift):
    rng = np.random.default_rng(vocab)
    requests, beams = (2, 4) if keep > 64 else (8, 4)
    logits = 2.5 * rng.standard_normal((requests, beams, vocab))
    # Each beam's largest are in one of the rounds, and between beams they grow and fall from round to round.
    at = np.arange(vocab) // CHUNK
    for r in range(requests):
        for b in range(beams):
            logits[r, b] += np.take(rng.permutation(at[-1] + 1), at) * (r % 3)
    _check(k, logits, -20 * rng.random((requests, beams)), rows // (requests * beams), keep, dtype, rounds, pad, shift)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_equal_logits_over_rounds(k, dtype):
    """Too many that reach the bound: taken one after another, from all rounds."""
    rng = np.random.default_rng(81)
    logits = rng.integers(0, 3, (4, 2, 25000)).astype(np.float32)
    logits[1, 0] = -2.5
    logits[2, 1, :24990] = 1.0  # the largest at the very end
    logits[2, 1, 24990:] = 4.0
    logits[3, 0, :20000] = -np.inf
    got = _check(k, logits, [[0, -7], [-3, -1.5], [-1, -1], [-2, -2]], 256, 40, dtype, 4)
    assert got[2][0, 1, :3].tolist() == got[2][255, 1, :3].tolist()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_what_takes_no_part_in_a_later_round(k, dtype):
    rng = np.random.default_rng(82)
    logits = rng.standard_normal((6, 2, 25000))
    logits[0, 0, 24999] = np.nan
    logits[0, 1, 8200] = np.nan
    logits[1, 0, 17000] = np.inf
    logits[1, 1, :24000] = -np.inf  # all but the last round
    logits[2, 0, 9000:] = -np.inf   # all but the first and a little
    logits[2, 1] = -np.inf
    logits[3, 0, 20000] = 1e30      # one that outweighs what came before
    logits[3, 1, 3] = 1e30
    logits[4, :, 5:24995] = -np.inf  # fewer than are kept
    scores = -rng.random((6, 2))
    scores[5] = (-np.inf, np.nan)
    got = _check(k, logits, scores, 171, 12, dtype, 4)
    assert (got[1][:, 5] == NONE).all() and (got[1][:, 0] == NONE).all()


def test_a_long_sum_of_equal_terms(k):
    """32 rounds in which each thread has one 1 and terms a little below it: added to one running sum in 32 bits, each
    would be rounded up to 1 from 512 terms on, 2^-16.1 of the sum in all."""
    vocab, rows = 32 * CHUNK, 2048
    assert _rounds(rows, vocab) == 32
    near = bf16(np.float32([-2.75e-5]))[0]
    row = np.full((1, 1, vocab), near, np.uint16)
    row[0, 0, :2048:8] = 0  # the first of each thread's first eight
    _say("select_beams: 32 rounds of nearly equal logits")
    got = _select(k, row, np.zeros((1, 1)), rows, 3, "bf16")
    x = f64(np.asarray([near]))[0]
    total = -np.log(256.0 + (vocab - 256) * np.exp(x))
    assert (got[2] == np.asarray([0, 8, 16], np.uint32)).all()
    error = np.abs(got[0] - total)
    _say(f"beams: largest error {error.max():.3g}, bound {2.0 ** -17 + 2.0 ** -24 * abs(total):.3g}")
    assert (error <= 2.0 ** -17 + 2.0 ** -24 * abs(total)).all()
