"""GPU tests of select_beams against the 64-bit restatement in
branch_reference.py. Parents and tokens are compared exactly: the scores of two
beams differ by more here than the sums' rounding (each of the sums of at most
524,288 exponentials, 32 bits a thread and wave, is off by less than 2^-17 of
itself: 32 roundings of 2^-24 a thread, 14 of the joins, and 2^-20 for each
exponential that counts, whose argument is above -22; so is its logarithm,
absolutely) unless a test makes them equal. Scores: 2^-17 for the sum, and half a
step of fp32, 2^-24 of the score."""
import numpy as np
import pytest

import sgl_rocm_kv as kv
from branch_reference import NONE, best_beams
from selection_reference import bf16, f64
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


class Case:
    """logits: float32 [request][beam][vocab]; pad: elements of anything between rows; shift: elements before the first."""

    def __init__(self, logits, scores, keep, dtype, pad=0, shift=0):
        self.requests, self.beams, self.vocab = logits.shape
        self.keep, self.dtype, self.shift = keep, dtype, shift
        raw = bf16(logits) if dtype == "bf16" else np.asarray(logits, np.float32)
        self.logits = f64(raw) if dtype == "bf16" else raw.astype(np.float64)
        self.scores = np.asarray(scores, np.float32)
        stride = self.vocab + pad
        flat = np.full(shift + self.requests * self.beams * stride, 0x7FC0 if dtype == "bf16" else np.nan, raw.dtype)
        flat[shift:].reshape(-1, stride)[:, :self.vocab] = raw.reshape(-1, self.vocab)
        flat = flat[:len(flat) - pad] if pad else flat  # the last row has nothing behind it
        self.plan = kv.BeamPlan.new(request_count=self.requests, beam_count=self.beams, vocab_size=self.vocab, max_kept=keep,
                                    dtype=dtype, row_stride=stride if pad else 0)
        out = 4 * self.requests * keep
        self.given = dict(logits=hip.DeviceBuffer.from_array(flat), logits_offset=shift * raw.itemsize,
                          scores=hip.DeviceBuffer.from_array(self.scores), best_scores=_filled(out + 64),
                          best_parents=_filled(out + 64), best_tokens=_filled(out + 64),
                          workspace=_filled(self.plan.workspace_required_bytes + 64, 0xFF))

    def run(self, k, stream=None):
        k.select_beams(self.plan, kv.BeamBuffers(**self.given), stream=stream)
        hip.synchronize()
        got = []
        for name, dtype in (("best_scores", np.float32), ("best_parents", np.uint32), ("best_tokens", np.uint32)):
            raw = self.given[name].download()
            n = 4 * self.requests * self.keep
            assert (raw[n:] == 0xA5).all()
            got.append(raw[:n].view(dtype).reshape(self.requests, self.keep))
        assert (self.given["workspace"].download()[self.plan.workspace_required_bytes:] == 0xFF).all()
        return got

    def check(self, k):
        got, want = self.run(k), best_beams(self.logits, self.scores.astype(np.float64), self.keep)
        k.check_errors()
        assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
        has = want[1] != NONE
        assert np.isneginf(got[0][~has]).all()
        error, bound = np.abs(got[0][has] - want[0][has]), 2.0 ** -17 + 2.0 ** -24 * np.abs(want[0][has])
        if has.any():
            _say(f"beams: largest error {error.max():.3g}, {(error / bound).max():.3f} of the bound")
        assert (error <= bound).all()
        return got


def _random(seed, requests, beams, vocab, keep, dtype, spread=2.5, **more):
    rng = np.random.default_rng(seed)
    return Case(spread * rng.standard_normal((requests, beams, vocab)), -20 * rng.random((requests, beams)), keep, dtype, **more)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("requests,beams,vocab,keep,pad,shift", [
    (1, 1, 1, 1, 0, 0), (1, 1, 1, 5, 0, 0), (2, 3, 2, 9, 0, 0), (3, 4, 63, 8, 0, 0), (1, 4, 8191, 8, 0, 0),
    (2, 4, 8192, 8, 0, 0), (2, 4, 8193, 8, 0, 0), (3, 5, 50257, 10, 47, 0), (2, 2, 50257, 4, 0, 1), (2, 2, 20001, 4, 3, 3),
    (1, 8, 128256, 16, 0, 0), (1, 2, 524288, 3, 0, 0), (2, 64, 300, 128, 0, 0), (2, 65, 200, 70, 1, 0),
    (1, 1024, 40, 100, 0, 0), (130, 2, 100, 4, 0, 0), (1, 1, 20000, 128, 0, 0), (2, 7, 9000, 33, 7, 5)])
def test_against_the_definition(k, dtype, requests, beams, vocab, keep, pad, shift):
    _say(f"select_beams {requests}x{beams}x{vocab} keep={keep} {dtype} pad={pad} shift={shift}")
    _random(vocab + keep, requests, beams, vocab, keep, dtype, pad=pad, shift=shift).check(k)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab,keep", [(300, 128), (40000, 128), (9000, 8), (20000, 40)])
def test_equal_logits_go_to_the_lower_token(k, dtype, vocab, keep):
    rng = np.random.default_rng(vocab)
    x = rng.integers(0, 3, (2, 3, vocab)).astype(np.float32)
    Case(x, [[0, -7, -50], [-3, -1.5, -90]], keep, dtype).check(k)
    Case(np.full((1, 1, vocab), -2.5), [[1.0]], keep, dtype).check(k)
    zeros = np.where(rng.random((1, 1, vocab)) < 0.5, 0.0, -0.0)
    Case(zeros, [[0.0]], keep, dtype).check(k)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_equal_beams_go_to_the_lower_beam(k, dtype):
    rng = np.random.default_rng(41)
    row = rng.standard_normal(30000)
    got = Case(np.broadcast_to(row, (2, 4, 30000)), [[-1, -1, -1, -1], [-2, -1, -1, -2]], 10, dtype).check(k)
    assert got[1][0, :4].tolist() == [0, 1, 2, 3] and got[1][1, :2].tolist() == [5, 6]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_what_takes_no_part(k, dtype):
    """Ended beams, masked tokens, and logits that are no numbers."""
    rng = np.random.default_rng(42)
    x = rng.standard_normal((6, 4, 9000))
    scores = -rng.random((6, 4))
    scores[0, 1:] = -np.inf                      # a prompt's first step
    scores[1] = -np.inf                          # nothing goes on
    scores[2, 0], scores[2, 2] = np.nan, np.inf
    x[3, 0, 17], x[3, 1, 8999], x[3, 2, 5] = np.nan, np.inf, -np.inf
    x[4, :, 3:] = -np.inf                        # fewer continuations than are kept
    x[4, 2] = -np.inf
    x[5, 0] = -np.inf
    x[5, 1, :8192] = -np.inf                     # a whole split
    x[5, 2, 1:] = -np.inf
    x[5, 3] = np.where(np.arange(9000) % 2, -np.inf, 3e38)
    got = Case(x, scores, 12, dtype).check(k)
    assert (got[1][1] == NONE).all() and (got[1][0] == 0).all() and (got[1][4] != NONE).sum() == 9


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_magnitudes(k, dtype):
    """Large logits, a wide spread, one that outweighs all, and scores far apart."""
    rng = np.random.default_rng(43)
    x = np.stack([3e4 * rng.standard_normal((2, 20000)), 1e-3 * rng.standard_normal((2, 20000)),
                  np.where(np.arange(40000).reshape(2, -1) % 20000 == 777, 1e30, -1e30), 1e38 * rng.standard_normal((2, 20000))])
    Case(x, [[-1000, 0], [0, -1e-3], [-5, -5.5], [0, 0]], 6, dtype).check(k)


def test_refusals(k):
    case = _random(44, 2, 3, 100, 4, "bf16")
    sizes = dict(logits=600 * 2, scores=24, best_scores=32, best_parents=32, best_tokens=32,
                 workspace=case.plan.workspace_required_bytes)

    def refused(variant, name, **change):
        with pytest.raises(kv.KvError) as e:
            k.select_beams(case.plan, kv.BeamBuffers(**{**case.given, **change}))
        assert (e.value.variant, e.value.name) == (variant, name)

    for name, n in sizes.items():
        refused("AllocationOutOfBounds", name, **{name: kv.device_buffer(case.given[name].ptr, n - 1)})
        refused("DeviceMismatch", name, **{name: kv.device_buffer(1 << 20, 1 << 30)})
    refused("InvalidArgument", "alignment", logits_offset=0, logits=kv.device_buffer(case.given["logits"].ptr + 1, 1 << 20))
    case.plan._c.config.dtype = 3
    refused("InvalidArgument", "dtype")
