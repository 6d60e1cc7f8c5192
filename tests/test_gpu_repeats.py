"""GPU tests that attention over staged rows repeats itself: the same call, back to back with another one, gives the
same bits every time. Everything that these kernels do has one order (no atomics on floats), so that any difference
is a wait that is missing or a row that was read too soon."""
import numpy as np
import pytest

import sgl_rocm_kv as kv
from branch_reference import Trees
from selection_reference import Batch, Pool
from sgl_rocm_kv import hip
from test_gpu_selection import _filled, _say

pytestmark = pytest.mark.gpu

ROUNDS = 12


@pytest.fixture(scope="module")
def k():
    if hip.device_count() == 0:
        pytest.fail("no GPU visible: the gpu tests need an MI355X")
    ctx = kv.RocmKvPairCopyKernels(0)
    yield ctx
    ctx.close()


def _repeats(calls, outputs):
    """calls[0], calls[1], calls[0], ... without a wait between them."""
    want = None
    for _ in range(ROUNDS):
        for b in outputs:
            b.upload(np.full(b.nbytes, 0xA5, np.uint8))
        hip.synchronize()
        for call in (calls[0], calls[1], calls[0]):
            call()
        hip.synchronize()
        got = [b.download() for b in outputs]
        if want is None:
            want = got
        differing = [int((g.view(np.uint16) != w.view(np.uint16)).sum()) for g, w in zip(got, want)]
        assert differing == [0, 0], differing


LONG = (8192, 7000, 300, 4111, 5000, 640, 2999, 8000, 1700, 3500, 6100, 900)


@pytest.mark.parametrize("shape", [
    dict(contexts=LONG, drafts=(24, 9, 16, 20, 12, 24, 8, 17, 23, 11, 13, 24)),          # four row waves
    dict(contexts=LONG, drafts=(7, 8, 6, 8, 5, 8, 8, 7, 8, 8, 6, 8), heads=8, qheads=32),  # two
    dict(contexts=(8192, 3000), drafts=(4, 5)),                                           # one
    dict(contexts=LONG[:6], drafts=(120, 100, 77, 60, 120, 99), words=2, hnd=True),
    dict(contexts=LONG, drafts=(61,) * 12, dk=64, qheads=14, hnd=True),
    dict(contexts=(5000,), drafts=(16,), dk=64),
    dict(contexts=LONG[:6], drafts=(16, 13, 9, 16, 2, 11), dk=256),
    dict(contexts=(3000,), drafts=(6,), dk=256),
    dict(contexts=(2000, 900), drafts=(16, 7), dk=40),                                    # the generic body
], ids=lambda s: f"dk{s.get('dk', 128)}-{len(s['contexts'])}x{max(s['drafts'])}-heads{s.get('heads', 2)}")
def test_tree_attention_repeats(k, shape):
    shape = {**dict(heads=2, qheads=8, dk=128, words=None, hnd=False), **shape}
    _say(f"tree attention repeats: {shape}")
    rng = np.random.default_rng(1)
    calls, outputs, held = [], [], []
    for _ in range(2):
        pages = sum(-(-(c + n) // 64) for c, n in zip(shape["contexts"], shape["drafts"])) + 2
        pool = Pool(rng, page=64, heads=shape["heads"], dk=shape["dk"], pages=pages, hnd=shape["hnd"], layers=2)
        trees = Trees(rng, pool, shape["qheads"], shape["contexts"], shape["drafts"], words=shape["words"])
        plan = trees.plan(max(c + n for c, n in zip(shape["contexts"], shape["drafts"])))
        output = _filled(plan.attention.output_required_bytes)
        buffers = kv.TreeAttentionBuffers(**trees.upload(), pool=pool.buffer, output=output,
                                          workspace=_filled(max(16, plan.workspace_required_bytes), 0xFF))
        held.append((trees, plan, buffers))
        outputs.append(output)
        calls.append(lambda plan=plan, buffers=buffers: k.tree_attention(plan, buffers))
    _repeats(calls, outputs)
    k.check_errors()


@pytest.mark.parametrize("dk,hnd,per", [(128, False, 1), (128, True, 1), (128, False, 100), (64, True, 1), (64, False, 100),
                                        (256, False, 1), (256, True, 60)])
def test_paged_attention_repeats(k, dk, hnd, per):
    """Single queries (staged rows) and prompts (tiles)."""
    _say(f"paged attention repeats: dk={dk} hnd={hnd} per={per}")
    rng = np.random.default_rng(2)
    calls, outputs, held = [], [], []
    for _ in range(2):
        pool = Pool(rng, page=64, heads=2, dk=dk, pages=sum(-(-n // 64) for n in LONG) + 2, hnd=hnd, layers=2)
        batch = Batch(rng, pool, LONG, 8, per=per)
        plan = batch.plan()
        output = _filled(plan.output_required_bytes)
        held.append((pool, batch))
        outputs.append(output)
        calls.append(lambda plan=plan, batch=batch, pool=pool, output=output: k.paged_attention_async(
            plan, **batch.device, pool=pool.buffer, output=output))
    _repeats(calls, outputs)
    k.check_errors()
