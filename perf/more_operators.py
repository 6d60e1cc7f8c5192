"""Decoding a request along several continuations over a paged KV cache, as cases that can be timed and checked: trees of
drafted tokens that are verified in one step, and beams that share their pages.

A case is a dict of plain values. ``op`` names the operator:

  tree   attention of drafted tokens over their request's tokens and their own ancestors (tree_attention)
  keep   the accepted drafts' rows moved together inside the cache, all layers (keep_drafts)
  beams  the best continuations of each request over its beams and the vocabulary (select_beams)
  fork   beams that go on from the chosen ones: shared pages, copied last pages, freed pages (fork_sequences)

With ``own`` false each is computed from elementary torch operations; with ``own`` true through the package's binding.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_GOLDEN = 0.6180339887498949
_LAYERS, _LAYER = 2, 1  # attention: a pool of two layers, of which the second is attended
_context = None


def _kv():
    """The package's binding and one context a process, as a serving program keeps it."""
    global _context
    if _context is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sglang-rs_amd"))
        import sgl_rocm_kv as kv
        _context = (kv, kv.RocmKvPairCopyKernels(0))
    return _context


# ---- the listed cases -----------------------------------------------------------------------


def listed():
    llama8b = dict(qheads=32, heads=8, dim=128, page=64, hnd=False)
    return [
        # One user's verification step: a tree of 16 drafted tokens. Latency counts.
        dict(name="tree_one_2048x16", op="tree", requests=1, low=2048, high=2048, drafts=16, words=1, **llama8b),
        # A serving batch of ragged contexts, up to 24 drafted tokens each.
        dict(name="tree_32x24", op="tree", requests=32, low=300, high=8192, drafts=24, words=1, **llama8b),
        # Wide trees of a small model (7 query heads a KV head, dims 64) over head-major 16-token pages.
        dict(name="tree_hnd64_24x61", op="tree", requests=24, low=700, high=6000, drafts=61, words=1, qheads=14, heads=2,
             dim=64, page=16, hnd=True),
        # Few requests with long contexts and trees of over a hundred tokens: two mask words.
        dict(name="tree_long_6x120", op="tree", requests=6, low=9000, high=32768, drafts=120, words=2, **llama8b),
        # A small model's few requests (24 layers, 2 KV heads of 64 dims): three or so rows each.
        dict(name="keep_hnd64_3", op="keep", requests=3, layers=24, drafts=16, kept=6, heads=2, dim=64, page=16, hnd=True),
        # A serving batch after a verification step, 32 layers.
        dict(name="keep_64x8", op="keep", requests=64, layers=32, drafts=32, kept=8, heads=8, dim=128, page=16, hnd=False),
        # One user's beams.
        dict(name="beams_one_4", op="beams", requests=1, beams=4, vocab=32000, keep=8, f32=False, pad=0),
        # A batch over an odd vocabulary, 32-bit logits whose rows are padded.
        dict(name="beams_f32_24x5", op="beams", requests=24, beams=5, vocab=50257, keep=10, f32=True, pad=47),
        # The largest batch: 256 rows of a large vocabulary.
        dict(name="beams_64x4", op="beams", requests=64, beams=4, vocab=128256, keep=8, f32=False, pad=0),
        # One user's beams change places: a page or two to copy.
        dict(name="fork_one_4", op="fork", requests=1, beams=4, low=500, high=500, layers=24, heads=2, dim=64, page=16,
             hnd=False, finished=0),
        # Head-major pages, odd counts, some requests finished.
        dict(name="fork_hnd_11x5", op="fork", requests=11, beams=5, low=40, high=900, layers=24, heads=2, dim=64, page=32,
             hnd=True, finished=2),
        # A batch of 256 beams (16 layers, 8 KV heads of 64 dims), 64-token pages.
        dict(name="fork_64x4", op="fork", requests=64, beams=4, low=90, high=700, layers=16, heads=8, dim=64, page=64,
             hnd=False, finished=3),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case over the range that the listed ones span, never above the largest of its operator."""
    case = _draw(rng)
    most = {k: max(_size(c)[k] for c in listed() if c["op"] == case["op"]) for k in ("bytes", "flops")}
    while any(_size(case)[k] > most[k] for k in most):
        if case["requests"] > 1:
            case["requests"] = case["requests"] * 2 // 3
            if "finished" in case:
                case["finished"] = min(case["finished"], case["requests"] // 2)
        elif "high" in case:
            case.update(high=case["high"] // 2, low=max(1, case["low"] // 2))
        else:
            case["beams"] -= 1
    return case


def _size(case):
    """work(), and for the page operators the pool that the case needs."""
    size = work(case)
    if case["op"] == "fork":
        size["bytes"] = _fork_pages(case)[3] * _token_bytes(case) * case["page"]
    return size


def _draw(rng):
    op = rng.choice(["tree", "tree", "tree", "keep", "beams", "beams", "fork", "fork"])
    if op == "beams":
        beams = rng.randint(1, 8)
        return dict(op=op, requests=_log(rng, 1, 64), beams=beams, vocab=_log(rng, 400, 152000),
                    keep=beams * rng.choice([1, 2, 2, 3]), f32=rng.random() < 0.4, pad=rng.choice([0, 0, 1, 8, 47]))
    qheads, heads, dim = rng.choice([(32, 8, 128), (14, 2, 64), (32, 8, 64), (8, 2, 256), (8, 1, 128)])
    shape = dict(heads=heads, dim=dim, page=rng.choice([16, 32, 64]), hnd=rng.random() < 0.4)
    if op == "tree":
        high, drafts = _log(rng, 16, 32768), _log(rng, 1, 128)
        return dict(op=op, requests=_log(rng, 1, 64), low=max(1, high // rng.choice([1, 3, 12])), high=high, drafts=drafts,
                    words=-(-drafts // 64), qheads=qheads, **shape)
    shape["layers"] = rng.choice([16, 24, 32])
    if op == "keep":
        drafts = _log(rng, 2, 64)
        return dict(op=op, requests=_log(rng, 1, 64), drafts=drafts, kept=rng.randint(1, min(drafts, 12)), **shape)
    requests, high = _log(rng, 1, 64), _log(rng, 20, 1500)
    return dict(op=op, requests=requests, beams=rng.randint(2, 8), low=max(1, high // rng.choice([1, 2, 8])), high=high,
                finished=rng.randint(0, requests // 4), **shape)


# ---- inputs ---------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ragged(count, low, high):
    """`count` lengths spread evenly over [low, high], in a scattered order; the first is `high`."""
    return [low + round((high - low) * (1.0 - (i * _GOLDEN) % 1.0)) for i in range(count)]


def _device(values, dtype):
    return torch.from_numpy(np.ascontiguousarray(values, dtype=dtype)).to("cuda")


def _page_slots(g, lengths, page):
    """Each sequence's pages, scattered over a pool of just enough of them: (slot of every token, pages)."""
    need = [-(-n // page) for n in lengths]
    total = sum(need)
    at = torch.randperm(total, generator=g, device="cuda")
    first = np.concatenate([[0], np.cumsum(need)])
    logical = np.concatenate([first[i] * page + np.arange(n) for i, n in enumerate(lengths)])
    logical = torch.from_numpy(logical).to("cuda")
    return at[logical // page] * page + logical % page, total


def _offsets(lengths):
    return _device(np.concatenate([[0], np.cumsum(lengths)]), np.int64)


def _token_bytes(case):
    return case["layers"] * 2 * case["heads"] * case["dim"] * 2


def _pool(g, pages, layers, case):
    """bf16 [page][layer][K, V][the page's rows]."""
    pool = torch.empty(pages, layers, 2, case["page"] * case["heads"] * case["dim"], dtype=torch.bfloat16, device="cuda")
    return pool.normal_(generator=g)


def _buffer(t):
    return _kv()[0].device_buffer(t.data_ptr(), t.numel() * t.element_size())


def _view(case, pool, layer):
    kv = _kv()[0]
    h, d, page = case["heads"], case["dim"], case["page"]
    region = page * h * d * 2
    return kv.pool_view(pool.data_ptr(), pool.numel() * 2, page_size=page, page_stride_bytes=pool[0].numel() * 2,
                        page_count=pool.shape[0], tensor_offset=(2 * layer * region, (2 * layer + 1) * region),
                        row_bytes=h * d * 2, tensor_count=2, heads=h, head_layout=kv.HND if case["hnd"] else kv.NHD)


def _all_layers(case, pool):
    return dict(layer_count=case["layers"], layer_stride_bytes=2 * case["page"] * case["heads"] * case["dim"] * 2)


def prepare(case, seed):
    state = dict(_PREPARE[case["op"]](case, _generator(seed)), case=case)
    if own:
        _OWN_PREPARE[case["op"]](case, state)
    return state


def _tree_counts(case):
    """(tokens of each request before its drafts, its drafts: at least a third of the most, the last one all of them)."""
    contexts = _ragged(case["requests"], case["low"], case["high"])
    return contexts, _ragged(case["requests"], max(1, case["drafts"] // 3), case["drafts"])[::-1]


def _prepare_tree(case, g):
    contexts, drafts = _tree_counts(case)
    lengths = [c + n for c, n in zip(contexts, drafts)]
    slots, pages = _page_slots(g, lengths, case["page"])
    # Draft 0 is the tree's root; each other one's parent is among the few drafts before it, so that the tree is some
    # levels deep. A draft attends its ancestors and itself.
    most, words = case["drafts"], case["words"]
    step = torch.randint(1, max(2, most // 4), (case["requests"], most), generator=g, device="cuda")
    masks = torch.zeros(case["requests"], most, words, dtype=torch.int64, device="cuda")
    for i in range(most):
        if i:
            parent = (i - step[:, i]).clamp(min=0)
            masks[:, i] = masks.gather(1, parent[:, None, None].expand(-1, 1, words))[:, 0]
        masks[:, i, i // 64] |= (1 << (i % 64)) - (1 << 64 if i % 64 == 63 else 0)
    live = torch.arange(most, device="cuda") < _device(drafts, np.int64)[:, None]
    queries = torch.empty(sum(drafts), case["qheads"], case["dim"], dtype=torch.bfloat16, device="cuda")
    return dict(contexts=_device(np.repeat(contexts, drafts), np.int64), requests=_device(np.repeat(np.arange(len(drafts)), drafts), np.int32),
                offsets=_offsets(lengths), slots=slots, masks=masks[live], pool=_pool(g, pages, _LAYERS, case), pages=pages,
                queries=queries.normal_(generator=g), lengths=lengths, drafts=drafts,
                output=torch.zeros(sum(drafts), case["qheads"], case["dim"], dtype=torch.bfloat16, device="cuda"))


def _keep_counts(case):
    """(drafts kept of each request, tokens before them)."""
    kept = _ragged(case["requests"], 1, case["kept"])
    return kept, _ragged(case["requests"], 1, 2 * case["page"] - 1)[::-1]


def _prepare_keep(case, g):
    kept, contexts = _keep_counts(case)
    slots, pages = _page_slots(g, [c + case["drafts"] for c in contexts], case["page"])
    # An accepted path: the root, then drafts further on in the tree.
    rank = torch.empty(case["requests"], case["drafts"], device="cuda").uniform_(generator=g)
    rank[:, 0] = 2.0
    best = torch.topk(rank, case["kept"], dim=1).indices
    at = torch.arange(case["kept"], device="cuda")
    live = at < _device(kept, np.int64)[:, None]
    chosen = torch.where(live, best, 1 << 30).sort(dim=1).values
    return dict(contexts=_device(contexts, np.int64), offsets=_offsets([c + case["drafts"] for c in contexts]), slots=slots,
                kept=torch.where(live, chosen, -1).to(torch.int32), pool=_pool(g, pages, case["layers"], case))


def _prepare_beams(case, g):
    rows = case["requests"] * case["beams"]
    dtype = torch.float32 if case["f32"] else torch.bfloat16
    logits = torch.empty(rows, case["vocab"] + case["pad"], device="cuda").normal_(generator=g) * 2.5
    scores = -20.0 * torch.empty(case["requests"], case["beams"], device="cuda").uniform_(generator=g)
    out = dict(best_scores=torch.zeros(case["requests"], case["keep"], device="cuda"))
    for name in ("parents", "tokens"):
        out["best_" + name] = torch.zeros(case["requests"], case["keep"], dtype=torch.int32, device="cuda")
    return dict(logits=logits.to(dtype), scores=scores, **out)


def _fork_lengths(case):
    """Each request's tokens: never whole pages, so that each beam's last page is its own. (A next token that begins a page
    would take one more at each of a state's passes, whose lengths stay.)"""
    page = case["page"]
    return [n if n % page else n + 1 for n in _ragged(case["requests"], case["low"], case["high"])]


def _fork_pages(case):
    """(pages that a request's beams share, full pages of each beam alone, pages of a sequence, pages of the pool)."""
    full = [n // case["page"] for n in _fork_lengths(case)]
    shared = [(2 * n + 2) // 3 for n in full]
    rows = [n - s for n, s in zip(full, shared)]
    held = sum(s + case["beams"] * (m + 1) for s, m in zip(shared, rows))
    return shared, rows, max(full) + 1, held + case["requests"] * case["beams"] + 3


def _prepare_fork(case, g):
    r, b, page = case["requests"], case["beams"], case["page"]
    lengths, (shared, rows, most, total) = _fork_lengths(case), _fork_pages(case)
    number = np.full((r, b, most), -1, np.int64)
    references = []
    for i in range(r):  # pages in order, scattered over the pool below
        first = len(references)
        number[i, :, :shared[i]] = first + np.arange(shared[i])
        alone = first + shared[i] + np.arange(b * (rows[i] + 1)).reshape(b, -1)
        number[i, :, shared[i]:shared[i] + rows[i] + 1] = alone
        references += [b] * shared[i] + [1] * alone.size
    at = torch.randperm(total, generator=g, device="cuda")
    number = torch.from_numpy(number.reshape(r * b, most)).to("cuda")
    tables = torch.where(number >= 0, at[number.clamp(min=0)], -1).to(torch.int32)
    held = len(references)
    counts = torch.zeros(total, dtype=torch.int32, device="cuda")
    counts[at[:held]] = _device(references, np.int32)
    free = torch.zeros(total, dtype=torch.int32, device="cuda")
    free[:total - held] = at[held:].to(torch.int32)
    # Each beam goes on from one of its request's; the last requests are finished.
    parents = torch.randint(0, b, (r, b), generator=g, device="cuda") + b * torch.arange(r, device="cuda")[:, None]
    parents[r - case["finished"]:] = -1
    lengths = _device(np.repeat(lengths, b), np.int64)
    return dict(parents=parents.reshape(-1).to(torch.int32), lengths=[lengths, torch.zeros_like(lengths)],
                tables=[tables, torch.full_like(tables, -1)], references=counts, free=free,
                free_count=_device([total - held], np.int64), pool=_pool(g, total, case["layers"], case), turn=0)


_PREPARE = dict(tree=_prepare_tree, keep=_prepare_keep, beams=_prepare_beams, fork=_prepare_fork)


# ---- the package's calls --------------------------------------------------------------------

_APPEND = 1  # tokens that each beam is about to write


def _workspace(s, plan):
    s["workspace"] = torch.empty(max(16, plan.workspace_required_bytes), dtype=torch.uint8, device="cuda")
    return _buffer(s["workspace"])


def _own_tree(case, s):
    kv = _kv()[0]
    h, d, page = case["heads"], case["dim"], case["page"]
    token = _LAYERS * 2 * h * d * 2
    layout = kv.PagedKvCacheLayout.new(kv.KvCacheRuntimeLayout("bf16", page, _LAYERS, h, d, 2, token, token * page), s["pages"])
    plan = kv.PagedAttentionPlan.for_layer(layout, _LAYER, len(s["requests"]), case["requests"], s["slots"].numel(),
                                           case["qheads"], d ** -0.5, kv.HND if case["hnd"] else kv.NHD)
    s["plan"] = kv.TreeAttentionPlan.new(plan, mask_words=case["words"], max_sequence_length=max(s["lengths"]))
    s["buffers"] = kv.TreeAttentionBuffers(
        queries=_buffer(s["queries"]), query_request_indices=_buffer(s["requests"]),
        query_sequence_lengths=_buffer(s["contexts"]), request_slot_offsets=_buffer(s["offsets"]),
        sequence_slots=_buffer(s["slots"]), pool=_buffer(s["pool"]), output=_buffer(s["output"]), masks=_buffer(s["masks"]),
        workspace=_workspace(s, s["plan"]))


def _own_keep(case, s):
    kv = _kv()[0]
    s["plan"] = kv.DraftPlan.new(request_count=case["requests"], sequence_slot_count=s["slots"].numel(), max_kept=case["kept"])
    s["buffers"] = kv.DraftBuffers(request_lengths=_buffer(s["contexts"]), request_slot_offsets=_buffer(s["offsets"]),
                                   sequence_slots=_buffer(s["slots"]), kept=_buffer(s["kept"]))
    s["view"] = _view(case, s["pool"], 0)


def _own_beams(case, s):
    kv = _kv()[0]
    s["plan"] = kv.BeamPlan.new(request_count=case["requests"], beam_count=case["beams"], vocab_size=case["vocab"],
                                max_kept=case["keep"], row_stride=case["vocab"] + case["pad"],
                                dtype="f32" if case["f32"] else "bf16")
    s["buffers"] = kv.BeamBuffers(logits=_buffer(s["logits"]), scores=_buffer(s["scores"]),
                                  best_scores=_buffer(s["best_scores"]), best_parents=_buffer(s["best_parents"]),
                                  best_tokens=_buffer(s["best_tokens"]), workspace=_workspace(s, s["plan"]))


def _own_fork(case, s):
    kv = _kv()[0]
    sequences, table_pages = s["tables"][0].shape
    s["plan"] = kv.ForkPlan.new(sequence_count=sequences, parent_count=sequences, table_pages=table_pages,
                                page_size=case["page"], page_count=s["pool"].shape[0], append_tokens=_APPEND)
    workspace = _workspace(s, s["plan"])
    s["buffers"] = [kv.ForkBuffers(
        parents=_buffer(s["parents"]), lengths=_buffer(s["lengths"][i]), page_tables=_buffer(s["tables"][i]),
        forked_lengths=_buffer(s["lengths"][1 - i]), forked_tables=_buffer(s["tables"][1 - i]),
        page_references=_buffer(s["references"]), free_pages=_buffer(s["free"]), free_count=_buffer(s["free_count"]),
        workspace=workspace) for i in (0, 1)]
    s["view"] = _view(case, s["pool"], 0)


_OWN_PREPARE = dict(tree=_own_tree, keep=_own_keep, beams=_own_beams, fork=_own_fork)


def _run_own(case, s):
    k, stream, op = _kv()[1], torch.cuda.current_stream().cuda_stream, case["op"]
    if op == "tree":
        k.tree_attention(s["plan"], s["buffers"], stream=stream)
        return s["output"]
    if op == "keep":
        k.keep_drafts(s["plan"], s["buffers"], s["view"], stream=stream, **_all_layers(case, s["pool"]))
        return s["pool"]
    if op == "beams":
        k.select_beams(s["plan"], s["buffers"], stream=stream)
        return [s["best_scores"], s["best_parents"], s["best_tokens"]]
    turn = s["turn"]
    k.fork_sequences(s["plan"], s["buffers"][turn], s["view"], stream=stream, **_all_layers(case, s["pool"]))
    s["turn"] = 1 - turn  # (the next step goes on from what this one wrote)
    return [s["lengths"][1 - turn], s["tables"][1 - turn], s["references"], s["free"], s["free_count"], s["pool"]]


# ---- the plain forms ------------------------------------------------------------------------


def _rows(case, pool):
    """The pool's rows: a view [page, layer, K and V, position, head, dim]."""
    h, d, page = case["heads"], case["dim"], case["page"]
    if case["hnd"]:
        return pool.view(*pool.shape[:3], h, page, d).transpose(3, 4)
    return pool.view(*pool.shape[:3], page, h, d)


def _plain_tree(case, s):
    r, h, d, page = case["requests"], case["heads"], case["dim"], case["page"]
    g, longest, most = case["qheads"] // h, max(s["lengths"]), max(s["drafts"])
    at = torch.arange(longest, device="cuda")
    slots = s["slots"][(s["offsets"][:-1, None] + at).clamp(max=s["slots"].numel() - 1)]
    rows = _rows(case, s["pool"])[:, _LAYER]
    keys, values = (rows[slots // page, t, slots % page].float() for t in (0, 1))  # [request, token, head, dim]
    # Each request's drafts, padded to the most that one has.
    first = torch.searchsorted(s["requests"], torch.arange(r + 1, dtype=torch.int32, device="cuda"))
    number = first[:-1, None] + torch.arange(most, device="cuda")
    has, number = number < first[1:, None], number.clamp(max=len(s["requests"]) - 1)
    place = at - s["contexts"][number][..., None]  # of each token among the drafts: [request, query, token]
    bits = torch.gather(s["masks"][number], 2, (place.clamp(min=0) // 64).clamp(max=case["words"] - 1))
    live = (place < 0) | ((place < 64 * case["words"]) & ((bits >> (place.clamp(min=0) % 64)) & 1 == 1))
    live = (live & has[..., None]).repeat_interleave(g, dim=1)[:, None]  # [request, 1, query and head, token]
    queries = s["queries"][number].float() * d ** -0.5
    queries = queries.view(r, most, h, g, d).permute(0, 2, 1, 3, 4).reshape(r, h, most * g, d)
    weights = torch.matmul(queries, keys.permute(0, 2, 3, 1).contiguous()).masked_fill_(~live, -math.inf)
    weights = torch.exp(weights - weights.amax(dim=3, keepdim=True).clamp(min=-3e38))
    output = torch.matmul(weights, values.transpose(1, 2).contiguous()) / weights.sum(dim=3, keepdim=True).clamp(min=1e-37)
    output = output.view(r, h, most, g, d).permute(0, 2, 1, 3, 4).reshape(r, most, h * g, d)
    s["output"].copy_(output[has])
    return s["output"]


def _plain_keep(case, s):
    page, kept = case["page"], s["kept"].long()
    at = (s["offsets"][:-1] + s["contexts"])[:, None]
    moves = kept >= 0
    to = s["slots"][at + torch.arange(case["kept"], device="cuda")][moves]
    source = s["slots"][at + kept.clamp(min=0)][moves]
    rows = _rows(case, s["pool"])
    rows[to // page, :, :, to % page] = rows[source // page, :, :, source % page]
    return s["pool"]


def _plain_beams(case, s):
    r, vocab = case["requests"], case["vocab"]
    # In 64 bits: continuations of two beams may be as near to each other as the sums' rounding.
    x = s["logits"][:, :vocab].double().view(r, case["beams"], vocab)
    top = x.amax(dim=2, keepdim=True)
    total = s["scores"].double()[..., None] + (x - (top + torch.log(torch.exp(x - top).sum(dim=2, keepdim=True))))
    total = torch.where(total.isfinite(), total, -math.inf).view(r, -1)
    best = torch.sort(total, dim=1, descending=True, stable=True)
    some = min(case["keep"], total.shape[1])
    values, order = best.values[:, :some], best.indices[:, :some]
    has, first = values > -math.inf, case["beams"] * torch.arange(r, device="cuda")[:, None]
    s["best_scores"].fill_(-math.inf)[:, :some] = values.float()
    s["best_parents"].fill_(-1)[:, :some] = torch.where(has, first + order // vocab, -1).int()
    s["best_tokens"].fill_(-1)[:, :some] = torch.where(has, order % vocab, -1).int()
    return [s["best_scores"], s["best_parents"], s["best_tokens"]]


def _plain_fork(case, s):
    turn, page, total = s["turn"], case["page"], s["pool"].shape[0]
    lengths, tables = s["lengths"][turn], s["tables"][turn].long()
    sequences, most = tables.shape
    parents = s["parents"].long()
    begins, parent = parents >= 0, parents.clamp(min=0)
    length = torch.where(begins, lengths[parent], 0)
    full, pages = length // page, -(-length // page)
    need = torch.where(begins, -(-(length + _APPEND) // page), 0)
    at = torch.arange(sequences, device="cuda")
    again = ((parents == parents[:, None]) & (at < at[:, None])).any(dim=1)  # an earlier one has the same parent
    copies = begins & again & (length % page > 0)
    # Fresh pages from the end of the free list, sequence by sequence.
    fresh = copies + need - pages
    before = torch.cumsum(fresh, 0) - fresh
    j = torch.arange(most, device="cuda")
    old = tables[parent]
    number = torch.where(copies[:, None], j - full[:, None], j - pages[:, None])
    free_count = s["free_count"]
    taken = s["free"].long()[(free_count - 1 - before[:, None] - number).clamp(0, total - 1)]
    new = torch.where(j < pages[:, None], old, -1)
    new = torch.where((number >= 0) & (j < need[:, None]), taken, new)
    # The last pages' rows, before the copied pages take their places in the tables.
    source, to = old[at, full.clamp(max=most - 1)][copies], new[at, full.clamp(max=most - 1)][copies]
    rows = _rows(case, s["pool"])
    live = (torch.arange(page, device="cuda") < (length % page)[copies][:, None])[:, None, None, :, None, None]
    rows[to] = torch.where(live, rows[source], rows[to])
    # References by difference; pages that nothing holds any more go to the free list's end, ascending.
    held = (j < -(-lengths // page)[:, None]).reshape(-1)
    change = torch.zeros(total + 1, dtype=torch.int64, device="cuda")
    change.index_add_(0, torch.where(new >= 0, new, total).view(-1), torch.ones(new.numel(), dtype=torch.int64, device="cuda"))
    change.index_add_(0, torch.where(held, tables.view(-1), total), torch.full((new.numel(),), -1, dtype=torch.int64, device="cuda"))
    references = s["references"] + change[:total]
    freed = (s["references"] > 0) & (references == 0)
    left = free_count - fresh.sum()
    end = torch.where(freed, left + torch.cumsum(freed, 0) - 1, total)
    longer = torch.cat([s["free"], s["free"][:1]])
    longer[end] = torch.arange(total, dtype=torch.int32, device="cuda")
    s["free"].copy_(longer[:total])
    s["references"].copy_(references)
    s["free_count"].copy_(left + freed.sum())
    s["lengths"][1 - turn].copy_(length)
    s["tables"][1 - turn].copy_(new)
    s["turn"] = 1 - turn
    return [s["lengths"][1 - turn], s["tables"][1 - turn], s["references"], s["free"], s["free_count"], s["pool"]]


_PLAIN = dict(tree=_plain_tree, keep=_plain_keep, beams=_plain_beams, fork=_plain_fork)


def run(state):
    case = state["case"]
    return _run_own(case, state) if own else _PLAIN[case["op"]](case, state)


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    op = case["op"]
    if op == "beams":
        rows = case["requests"] * case["beams"]
        return dict(bytes=rows * (case["vocab"] * (4 if case["f32"] else 2) + 4) + 12 * case["requests"] * case["keep"],
                    flops=3.0 * rows * case["vocab"])
    if op == "tree":
        contexts, drafts = _tree_counts(case)
        rows, token = 2 * case["qheads"] * case["dim"], 4 * case["heads"] * case["dim"]
        seen = sum(n * c + min(n * n, n * (2 + math.log2(n))) for c, n in zip(contexts, drafts))  # (ancestors: about as many)
        return dict(bytes=2 * rows * sum(drafts) + token * (sum(contexts) + sum(drafts)) + 8 * case["words"] * sum(drafts),
                    flops=4.0 * case["qheads"] * case["dim"] * seen)
    if op == "keep":
        moved = sum(n - 1 for n in _keep_counts(case)[0])  # (the root stays; the drafts after it mostly move)
        return dict(bytes=2 * moved * _token_bytes(case) + 4 * case["requests"] * case["kept"], flops=0)
    # Of b children that choose their parents freely, b (1 - 1 / b)^b parents have none: as many last pages are copied.
    b, going = case["beams"], case["requests"] - case["finished"]
    copied = b * (1 - 1 / b) ** b * sum(n % case["page"] for n in _fork_lengths(case)[:going])
    return dict(bytes=2 * copied * _token_bytes(case) + 12 * case["requests"] * b * _fork_pages(case)[2], flops=0)


# ---- the definitions in 64 bits -------------------------------------------------------------


def exact(case, seed):
    """What run() returns, sequence by sequence and in 64 bits."""
    return _EXACT[case["op"]](case, _PREPARE[case["op"]](case, _generator(seed)))


def _slot_rows(case, pool, layer, tensor):
    """[slot, head, dim] of one layer's keys (0) or values (1)."""
    rows = pool[:, layer, tensor]
    h, d, page = case["heads"], case["dim"], case["page"]
    if case["hnd"]:
        rows = rows.reshape(-1, h, page, d).permute(0, 2, 1, 3)
    return rows.reshape(-1, h, d)


def _exact_tree(case, s):
    h, d = case["heads"], case["dim"]
    keys, values = (_slot_rows(case, s["pool"], _LAYER, t) for t in (0, 1))
    output = torch.zeros(s["output"].shape, dtype=torch.float64, device="cuda")
    masks, contexts = s["masks"].cpu().numpy().view(np.uint64), s["contexts"].tolist()
    first = 0
    for request, count in enumerate(s["drafts"]):
        begin, length = int(s["offsets"][request]), s["lengths"][request]
        slots = s["slots"][begin:begin + length]
        seen = np.zeros((count, length), bool)
        for i in range(count):
            context = contexts[first + i]
            seen[i, :context] = True
            tree = np.unpackbits(masks[first + i].view(np.uint8), bitorder="little")[:length - context]
            seen[i, context:context + len(tree)] = tree
        unseen = torch.from_numpy(~seen).to("cuda")[:, None]
        for k in range(h):
            mine = s["queries"][first:first + count].view(count, h, -1, d)[:, k].double()
            scores = (mine.reshape(-1, d) @ keys[slots, k].double().t().contiguous()).view(count, -1, length) * d ** -0.5
            weights = torch.softmax(scores.masked_fill_(unseen, -math.inf), dim=2)
            out = (weights.view(-1, length) @ values[slots, k].double()).view(count, -1, d)
            output[first:first + count].view(count, h, -1, d)[:, k] = out
        first += count
    return output


def _token_axis(case, pool, at, position):
    """A position of each of the pages `at`: the index of it in the pool's view by pages."""
    return (at, slice(None), slice(None), slice(None), position) if case["hnd"] else (at, slice(None), slice(None), position)


def _by_page(case, pool):
    h, d, page = case["heads"], case["dim"], case["page"]
    return pool.view(*pool.shape[:3], *((h, page, d) if case["hnd"] else (page, h, d)))


def _exact_keep(case, s):
    page, out = case["page"], s["pool"].double()
    rows, before = _by_page(case, out), _by_page(case, s["pool"])
    slots = s["slots"].tolist()
    for request, (begin, context) in enumerate(zip(s["offsets"].tolist(), s["contexts"].tolist())):
        for i, draft in enumerate(s["kept"][request].tolist()):
            if draft >= 0:
                to, source = slots[begin + context + i], slots[begin + context + draft]
                rows[_token_axis(case, out, to // page, to % page)] = before[_token_axis(case, out, source // page, source % page)].double()
    return out


def _exact_beams(case, s):
    rest = [], [], []
    for request in range(case["requests"]):
        row = s["logits"][request * case["beams"]:(request + 1) * case["beams"], :case["vocab"]].double()
        total = (s["scores"][request].double()[:, None] + torch.log_softmax(row, dim=1)).reshape(-1).cpu().numpy()
        total[~np.isfinite(total)] = -np.inf
        order = np.lexsort((np.arange(total.size), -total))[:case["keep"]]
        order = order[total[order] > -np.inf]
        fill = case["keep"] - len(order)
        rest[0].append(np.concatenate([total[order], np.full(fill, -np.inf)]))
        rest[1].append(np.concatenate([request * case["beams"] + order // case["vocab"], np.full(fill, -1)]))
        rest[2].append(np.concatenate([order % case["vocab"], np.full(fill, -1)]))
    return [torch.from_numpy(np.stack(x)) for x in rest[:1]] + [torch.from_numpy(np.stack(x).astype(np.int32)) for x in rest[1:]]


def _exact_fork(case, s):
    page, out = case["page"], s["pool"].double()
    rows, before = _by_page(case, out), _by_page(case, s["pool"])
    lengths, tables = s["lengths"][0].tolist(), s["tables"][0].tolist()
    free, references = s["free"].tolist(), s["references"].tolist()
    held = [r > 0 for r in references]
    end = int(s["free_count"])
    new_lengths, new_tables, seen = [], [], set()
    for p in s["parents"].tolist():
        table = [-1] * len(tables[0])
        length = lengths[p] if p >= 0 else 0
        for j in range(-(-(length + _APPEND) // page) if p >= 0 else 0):
            last = j == length // page and length % page > 0
            if j * page >= length or (last and p in seen):
                end -= 1
                table[j] = free[end]
                if last:
                    live = slice(0, length % page)
                    rows[_token_axis(case, out, table[j], live)] = before[_token_axis(case, out, tables[p][j], live)].double()
            else:
                table[j] = tables[p][j]
            references[table[j]] += 1
        seen.add(p)
        new_lengths.append(length)
        new_tables.append(table)
    for length, table in zip(lengths, tables):
        for j in range(-(-length // page)):
            references[table[j]] -= 1
    for number, (count, was) in enumerate(zip(references, held)):
        if was and count == 0:
            free[end] = number
            end += 1
    return [torch.tensor(new_lengths), torch.tensor(new_tables, dtype=torch.int32), torch.tensor(references, dtype=torch.int32),
            torch.tensor(free, dtype=torch.int32), torch.tensor([end]), out]


_EXACT = dict(tree=_exact_tree, keep=_exact_keep, beams=_exact_beams, fork=_exact_fork)
