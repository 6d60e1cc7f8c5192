"""Long-context operators over a paged bf16 KV cache, as cases that can be timed and checked: attention that reads only
the pages that a cheap score selects, and eviction of the tokens that got the least attention.

A case is a dict of plain values. ``op`` names the operator:

  bounds    each page's per-channel minimum and maximum of its keys (page_bounds)
  select    the pages of each (query, KV head) with the largest upper bound of q.k (select_pages)
  attend    softmax attention over each (query, KV head)'s own page list (selected_attention)
  weights   softmax weights of all queries added to each position's running sum (accumulate_weights)
  evict     the positions with the largest sums, and their K/V rows and sums copied out (select_tokens, compact_tokens)

With ``own`` false each is computed from elementary torch operations; with ``own`` true through the package's binding.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_GOLDEN = 0.6180339887498949
_LAYERS, _LAYER = 2, 1  # a pool of two layers; the operators work on the second
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
        # One decode step of 64 requests: the page that each one's new token went to. All launch and latency.
        dict(name="bounds_step_64", op="bounds", pages=64, total=4096, full=False, heads=8, dim=128, page=64, hnd=False),
        # All pages of prompts that were just written or received, head-major 16-token pages.
        dict(name="bounds_prompt_100000", op="bounds", pages=6250, total=8192, full=True, heads=8, dim=128, page=16, hnd=True),
        # One user's long context: 32 of 512 pages.
        dict(name="select_one_32768", op="select", requests=1, per=1, low=32768, high=32768, keep=32, **llama8b),
        # A decode batch of ragged long contexts in small pages: up to 2,048 pages a sequence.
        dict(name="select_page16_64", op="select", requests=64, per=1, low=3001, high=32768, keep=128,
             **dict(llama8b, page=16)),
        # Drafted tokens of a small model (7 query heads a KV head, dims 64), each with a list of its own.
        dict(name="select_verify_24x5", op="select", requests=24, per=5, low=700, high=20000, keep=48, qheads=14, heads=2,
             dim=64, page=16, hnd=True),
        # One user's step over 32 selected pages: 2,048 of 32,768 tokens.
        dict(name="attend_one_2048", op="attend", requests=1, per=1, low=32768, high=32768, keep=32, **llama8b),
        # The decode batch: 64 requests, 2,048 tokens each.
        dict(name="attend_64x2048", op="attend", requests=64, per=1, low=1000, high=16384, keep=32, **llama8b),
        # Drafted tokens over head-major 16-token pages, dims 256: pages end inside every tile.
        dict(name="attend_hnd256_24x5", op="attend", requests=24, per=5, low=300, high=8000, keep=45, qheads=8, heads=2,
             dim=256, page=16, hnd=True),
        # A decode step that keeps each position's attention sums, ragged up to 4,096 tokens.
        dict(name="weights_step_64", op="weights", requests=64, per=1, low=100, high=4096, **llama8b),
        # The sums of four ragged prompts, every prompt token a query.
        dict(name="weights_prompt_4", op="weights", requests=4, per=0, low=300, high=2048, **llama8b),
        # A few small-model requests cut to 1,000 tokens.
        dict(name="evict_hnd64_3", op="evict", requests=3, low=2500, high=5001, keep=1000, qheads=14, heads=2, dim=64,
             page=16, hnd=True),
        # A batch of long contexts cut to 2,048 tokens each.
        dict(name="evict_32x2048", op="evict", requests=32, low=2100, high=16384, keep=2048, **llama8b),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case over the range that the listed ones span, never above the largest of its operator."""
    case = _draw(rng)
    most = {k: max(work(c)[k] for c in listed() if c["op"] == case["op"]) for k in ("bytes", "flops")}
    size = "pages" if case["op"] == "bounds" else "requests"
    while any(work(case)[k] > most[k] for k in most):
        if case[size] > 1:
            case[size] = case[size] * 2 // 3
        else:
            case.update(high=case["high"] // 2, low=max(case.get("per", 1), 1, case["low"] // 2))
    return case


def _draw(rng):
    op = rng.choice(["bounds", "select", "select", "attend", "attend", "weights", "weights", "evict"])
    qheads, heads, dim = rng.choice([(32, 8, 128), (14, 2, 64), (32, 8, 64), (8, 2, 256), (8, 1, 128)])
    page, hnd = rng.choice([16, 32, 64]), rng.random() < 0.4
    shape = dict(heads=heads, dim=dim, page=page, hnd=hnd)
    if op == "bounds":
        pages = _log(rng, 1, 100000 * 8 * 128 // (page * max(heads * dim, 128)))
        return dict(op=op, pages=pages, total=pages + rng.randint(0, 500), full=rng.random() < 0.5, **shape)
    shape["qheads"] = qheads
    if op in ("select", "attend"):
        high = _log(rng, 1500, 32768) if op == "select" else _log(rng, 40, 16384)
        per, most = rng.choice([1, 1, 1, 5]), min(128, 2048 // page)
        if op == "select":  # (a list takes some of the longest sequence's pages)
            most = min(most, high // page // 3)
        return dict(op=op, requests=_log(rng, 1, 64 // per), per=per, low=max(per, high // rng.choice([1, 3, 10])),
                    high=high, keep=rng.randint(4, most), **shape)
    if op == "weights":
        if rng.random() < 0.3:
            high = _log(rng, 20, 2048)
            return dict(op=op, requests=rng.randint(1, 4), per=0, low=max(1, high // 8), high=high, **shape)
        per = rng.choice([1, 1, 3, 17])
        high = _log(rng, 40, 4096)
        return dict(op=op, requests=_log(rng, 1, 64 // per), per=per, low=max(per, high // rng.choice([1, 4, 16])),
                    high=high, **shape)
    high = _log(rng, 100, 16384)
    return dict(op=op, requests=_log(rng, 1, 32), low=max(1, high // rng.choice([1, 3, 8])), high=high,
                keep=_log(rng, 30, min(high, 2048)), **shape)


# ---- inputs ---------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ragged(count, low, high):
    """`count` lengths spread evenly over [low, high], in a scattered order; the first is `high`."""
    return [low + round((high - low) * (1.0 - (i * _GOLDEN) % 1.0)) for i in range(count)]


def _counts(case):
    """(tokens of each request, queries of each request)."""
    lengths = _ragged(case["requests"], case["low"], case["high"])
    return lengths, list(lengths) if case["per"] == 0 else [case["per"]] * len(lengths)


def _page_slots(g, lengths, page):
    """Each request's pages, scattered over a pool of just enough of them: (slot of every token, pages)."""
    need = [-(-n // page) for n in lengths]
    total = sum(need)
    at = torch.randperm(total, generator=g, device="cuda")
    first = np.concatenate([[0], np.cumsum(need)])
    logical = np.concatenate([first[i] * page + np.arange(n) for i, n in enumerate(lengths)])
    logical = torch.from_numpy(logical).to("cuda")
    return at[logical // page] * page + logical % page, total


def _metadata(lengths, counts):
    """Request and length of each query (a request's last ones, in order), and the requests' slot offsets."""
    requests = np.repeat(np.arange(len(counts)), counts)
    ends = np.concatenate([n - c + 1 + np.arange(c) for n, c in zip(lengths, counts)])
    return (torch.from_numpy(requests.astype(np.int32)).to("cuda"), torch.from_numpy(ends.astype(np.int64)).to("cuda"),
            torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to("cuda"))


def _pool(g, pages, case):
    """bf16 [page][layer][K, V][the page's rows]."""
    pool = torch.empty(pages, _LAYERS, 2, case["page"] * case["heads"] * case["dim"], dtype=torch.bfloat16, device="cuda")
    return pool.normal_(generator=g)


def _buffer(t):
    return _kv()[0].device_buffer(t.data_ptr(), t.numel() * t.element_size())


def _attention_plan(case, pages, queries, requests, slots):
    kv = _kv()[0]
    h, d, page = case["heads"], case["dim"], case["page"]
    token = _LAYERS * 2 * h * d * 2
    runtime = kv.KvCacheRuntimeLayout("bf16", page, _LAYERS, h, d, 2, token, token * page)
    layout = kv.PagedKvCacheLayout.new(runtime, pages)
    head_layout = kv.HND if case["hnd"] else kv.NHD
    return layout, kv.PagedAttentionPlan.for_layer(layout, _LAYER, queries, requests, slots, case["qheads"], d ** -0.5,
                                                   head_layout)


def _view(case, pool):
    kv = _kv()[0]
    h, d, page = case["heads"], case["dim"], case["page"]
    region = page * h * d * 2
    return kv.pool_view(pool.data_ptr(), pool.numel() * 2, page_size=page, page_stride_bytes=2 * _LAYERS * region,
                        page_count=pool.shape[0], tensor_offset=(2 * _LAYER * region, (2 * _LAYER + 1) * region),
                        row_bytes=h * d * 2, tensor_count=2, heads=h, head_layout=kv.HND if case["hnd"] else kv.NHD)


def prepare(case, seed):
    state = dict(_PREPARE[case["op"]](case, _generator(seed)), case=case)
    if own:
        _OWN_PREPARE[case["op"]](case, state)
    return state


def _prepare_bounds(case, g):
    n, total, page = case["pages"], case["total"], case["page"]
    pages = torch.randperm(total, generator=g, device="cuda")[:n].to(torch.int32)
    counts = torch.full((n,), page, dtype=torch.int32, device="cuda")
    if not case["full"]:
        counts = torch.randint(1, page + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
    return dict(pool=_pool(g, total, case), pages=pages, counts=counts,
                bounds=torch.zeros(total, case["heads"], 2, case["dim"], dtype=torch.bfloat16, device="cuda"))


def _prepare_sequences(case, g):
    lengths, counts = _counts(case)
    slots, pages = _page_slots(g, lengths, case["page"])
    requests, ends, offsets = _metadata(lengths, counts)
    queries = torch.empty(len(requests), case["qheads"], case["dim"], dtype=torch.bfloat16, device="cuda")
    return dict(slots=slots, pages=pages, requests=requests, ends=ends, offsets=offsets, lengths=lengths, counts=counts,
                queries=queries.normal_(generator=g), longest=max(lengths))


def _prepare_select(case, g):
    s = _prepare_sequences(case, g)
    # A page's keys lie around a centre of their own.
    shape = (s["pages"], case["heads"], case["dim"])
    centre = torch.empty(shape, device="cuda").normal_(generator=g) * 0.5
    low, high = (torch.empty(shape, device="cuda").normal_(generator=g).abs() + 1.0 for _ in range(2))
    s["bounds"] = torch.stack([centre - low, centre + high], dim=2).to(torch.bfloat16)
    s["selected"] = torch.zeros(len(s["requests"]), case["heads"], case["keep"], dtype=torch.int32, device="cuda")
    return s


def _prepare_attend(case, g):
    s = _prepare_sequences(case, g)
    s["pool"] = _pool(g, s["pages"], case)
    page, most = case["page"], -(-s["longest"] // case["page"])
    # Each (query, KV head) has pages of its own, the newest always among them.
    own_pages = (s["ends"] + page - 1)[:, None, None] // page
    rank = torch.empty(len(s["requests"]), case["heads"], most, device="cuda").uniform_(generator=g)
    at = torch.arange(most, device="cuda")
    rank = torch.where(at == own_pages - 1, 2.0, torch.where(at < own_pages, rank, -1.0))
    best = torch.topk(rank, min(case["keep"], most), dim=2)
    ids = torch.where(best.values >= 0, best.indices, 1 << 30).sort(dim=2).values
    ids = torch.nn.functional.pad(ids, (0, case["keep"] - ids.shape[2]), value=1 << 30)
    s["selected"] = torch.where(ids < 1 << 30, ids, -1).to(torch.int32)
    s["output"] = torch.zeros(len(s["requests"]), case["qheads"], case["dim"], dtype=torch.bfloat16, device="cuda")
    return s


def _prepare_weights(case, g):
    s = _prepare_sequences(case, g)
    s["pool"] = _pool(g, s["pages"], case)
    s["weights"] = torch.empty(case["heads"], sum(s["lengths"]), device="cuda").uniform_(generator=g)
    return s


def _prepare_evict(case, g):
    lengths = _ragged(case["requests"], case["low"], case["high"])
    slots, pages = _page_slots(g, lengths, case["page"])
    kept = [min(n, case["keep"]) for n in lengths]
    to_slots, to_pages = _page_slots(g, kept, case["page"])
    # Sums of softmax weights spread over decades.
    weights = torch.exp(3.0 * torch.empty(case["heads"], sum(lengths), device="cuda").normal_(generator=g))
    cumulated = [torch.tensor([0] + n, dtype=torch.int64).cumsum(0).to("cuda") for n in (lengths, kept)]
    return dict(lengths=torch.tensor(lengths, dtype=torch.int64, device="cuda"), offsets=cumulated[0], slots=slots,
                pool=_pool(g, pages, case), weights=weights, to_offsets=cumulated[1], to_slots=to_slots, tokens=sum(lengths),
                to_pool=torch.zeros(to_pages, *_pool(g, 0, case).shape[1:], dtype=torch.bfloat16, device="cuda"),
                to_weights=torch.zeros(case["heads"], sum(kept), device="cuda"), longest=max(lengths), to_tokens=sum(kept),
                kept=torch.zeros(len(lengths), case["heads"], case["keep"], dtype=torch.int32, device="cuda"))


# ---- the package's calls --------------------------------------------------------------------

_FORCED = dict(first_pages=1, last_pages=1)  # pages in every list: a prompt's start, and the newest tokens
_FORCED_TOKENS = dict(first_tokens=4, last_tokens=16)


def _own_bounds(case, s):
    s["view"] = _view(case, s["pool"])
    s["at"] = dict(pages=_buffer(s["pages"]), counts=_buffer(s["counts"]), bounds=_buffer(s["bounds"]))


def _attention_buffers(s):
    return dict(queries=_buffer(s["queries"]), query_request_indices=_buffer(s["requests"]),
                query_sequence_lengths=_buffer(s["ends"]), request_slot_offsets=_buffer(s["offsets"]),
                sequence_slots=_buffer(s["slots"]))


def _workspace(s, plan):
    s["workspace"] = torch.empty(max(16, plan.workspace_required_bytes), dtype=torch.uint8, device="cuda")
    return _buffer(s["workspace"])


def _own_selection(case, s):
    kv = _kv()[0]
    plan = _attention_plan(case, s["pages"], len(s["requests"]), case["requests"], s["slots"].numel())[1]
    forced = {k: min(v, case["keep"] // 2) for k, v in _FORCED.items()}
    s["plan"] = kv.PageSelectionPlan.new(plan, max_pages=case["keep"], max_sequence_length=s["longest"], **forced)
    named = dict(_attention_buffers(s), selected=_buffer(s["selected"]), workspace=_workspace(s, s["plan"]))
    if case["op"] == "select":
        named["bounds"] = _buffer(s["bounds"])
    else:
        named.update(pool=_buffer(s["pool"]), output=_buffer(s["output"]))
    s["buffers"] = kv.PageSelectionBuffers(**named)


def _own_weights(case, s):
    kv = _kv()[0]
    plan = _attention_plan(case, s["pages"], len(s["requests"]), case["requests"], s["slots"].numel())[1]
    s["plan"] = kv.WeightAccumulationPlan.new(plan, max_sequence_length=s["longest"])
    s["buffers"] = kv.WeightAccumulationBuffers(**_attention_buffers(s), pool=_buffer(s["pool"]),
                                                weights=_buffer(s["weights"]), workspace=_workspace(s, s["plan"]))


def _own_evict(case, s):
    kv = _kv()[0]
    s["plan"] = kv.EvictionPlan.new(request_count=case["requests"], kv_head_count=case["heads"],
                                    sequence_slot_count=s["tokens"], destination_slot_count=s["to_tokens"],
                                    max_kept=case["keep"], max_sequence_length=s["longest"], **_forced_tokens(case))
    s["buffers"] = kv.EvictionBuffers(
        request_lengths=_buffer(s["lengths"]), request_slot_offsets=_buffer(s["offsets"]),
        sequence_slots=_buffer(s["slots"]), weights=_buffer(s["weights"]), kept=_buffer(s["kept"]),
        destination_slot_offsets=_buffer(s["to_offsets"]), destination_slots=_buffer(s["to_slots"]),
        destination_weights=_buffer(s["to_weights"]), workspace=_workspace(s, s["plan"]))
    s["views"] = _view(case, s["pool"]), _view(case, s["to_pool"])


_PREPARE = dict(bounds=_prepare_bounds, select=_prepare_select, attend=_prepare_attend, weights=_prepare_weights,
                evict=_prepare_evict)
_OWN_PREPARE = dict(bounds=_own_bounds, select=_own_selection, attend=_own_selection, weights=_own_weights,
                    evict=_own_evict)


def _forced_tokens(case):
    return {k: min(v, case["keep"] // 2) for k, v in _FORCED_TOKENS.items()}


def _run_own(case, s):
    k, stream, op = _kv()[1], torch.cuda.current_stream().cuda_stream, case["op"]
    if op == "bounds":
        k.page_bounds(s["view"], page_count=case["pages"], stream=stream, **s["at"])
        return s["bounds"]
    if op == "select":
        k.select_pages(s["plan"], s["buffers"], stream=stream)
        return s["selected"]
    if op == "attend":
        k.selected_attention(s["plan"], s["buffers"], stream=stream)
        return s["output"]
    if op == "weights":
        k.accumulate_weights(s["plan"], s["buffers"], stream=stream)
        return s["weights"]
    k.select_tokens(s["plan"], s["buffers"], stream=stream)
    k.compact_tokens(s["plan"], s["buffers"], *s["views"], stream=stream)
    return [s["kept"], s["to_pool"], s["to_weights"]]


# ---- the plain forms ------------------------------------------------------------------------


def _rows(case, pool):
    """(keys, values) of the layer: views [page, position, head, dim] of the pool."""
    h, d, page = case["heads"], case["dim"], case["page"]
    layer = pool[:, _LAYER]
    if case["hnd"]:
        both = layer.view(-1, 2, h, page, d).transpose(2, 3)
    else:
        both = layer.view(-1, 2, page, h, d)
    return both[:, 0], both[:, 1]


def _plain_bounds(case, s):
    keys = _rows(case, s["pool"])[0][s["pages"].long()].float()
    live = (torch.arange(case["page"], device="cuda") < s["counts"][:, None])[:, :, None, None]
    low = torch.where(live, keys, math.inf).amin(dim=1)
    high = torch.where(live, keys, -math.inf).amax(dim=1)
    s["bounds"][s["pages"].long()] = torch.stack([low, high], dim=2).to(torch.bfloat16)
    return s["bounds"]


def _best(values, rank, keep):
    """Indices along the last axis of the `keep` first by (rank, larger value, lower index), ascending; -1 for those
    of rank 2."""
    order = torch.sort(values, dim=-1, descending=True, stable=True).indices
    by_rank = torch.sort(torch.gather(rank, -1, order), dim=-1, stable=True)
    order = torch.gather(order, -1, by_rank.indices)[..., :keep]
    order = torch.where(by_rank.values[..., :keep] < 2, order, 1 << 30).sort(dim=-1).values
    order = torch.nn.functional.pad(order, (0, keep - order.shape[-1]), value=1 << 30)
    return torch.where(order < 1 << 30, order, -1).to(torch.int32)


def _page_of(case, s, logical):
    """Pool page of each (query, ..., logical page); pages past the query's end give some page of the pool."""
    at = s["offsets"][s["requests"].long()].view(-1, *[1] * (logical.dim() - 1)) + logical.clamp(min=0) * case["page"]
    return s["slots"][at.clamp(max=s["slots"].numel() - 1)] // case["page"]


def _plain_select(case, s):
    most, page, h = -(-s["longest"] // case["page"]), case["page"], case["heads"]
    at = torch.arange(most, device="cuda")
    bounds = s["bounds"][_page_of(case, s, at.expand(len(s["requests"]), most))].double()  # [query, page, head, 2, dim]
    low, high = bounds[:, :, :, 0].permute(0, 2, 3, 1), bounds[:, :, :, 1].permute(0, 2, 3, 1)
    queries = s["queries"].view(len(s["requests"]), h, -1, case["dim"]).double()
    scores = torch.matmul(queries.clamp(min=0), high.contiguous()) + torch.matmul(queries.clamp(max=0), low.contiguous())
    scores = scores.amax(dim=2)
    pages = ((s["ends"] + page - 1) // page)[:, None, None]
    first, last = (min(v, case["keep"] // 2) for v in _FORCED.values())
    rank = torch.where((at < first) | (at >= pages - last), 0, 1)
    rank = torch.where(at < pages, rank, 2).expand_as(scores)
    s["selected"].copy_(_best(scores, rank, case["keep"]))
    return s["selected"]


def _plain_attend(case, s):
    n, h, page, d = len(s["requests"]), case["heads"], case["page"], case["dim"]
    selected = s["selected"].long()
    physical = _page_of(case, s, selected)
    heads = torch.arange(h, device="cuda")[None, :, None]
    keys, values = (x[physical, :, heads].float().reshape(n, h, -1, d) for x in _rows(case, s["pool"]))
    token = selected[..., None] * page + torch.arange(page, device="cuda")
    live = ((selected[..., None] >= 0) & (token < s["ends"][:, None, None, None])).reshape(n, h, 1, -1)
    queries = s["queries"].view(n, h, -1, d).float() * d ** -0.5
    scores = torch.matmul(queries, keys.transpose(2, 3)).masked_fill(~live, -math.inf)
    top = scores.amax(dim=3, keepdim=True)
    weights = torch.where(live, torch.exp(scores - top), 0.0)
    output = torch.matmul(weights, values) / weights.sum(dim=3, keepdim=True)
    s["output"].copy_(torch.where(live.any(dim=3, keepdim=True), output, 0.0).reshape(n, -1, d))
    return s["output"]


def _plain_weights(case, s):
    r, h, d, longest, most = case["requests"], case["heads"], case["dim"], s["longest"], max(s["counts"])
    g = case["qheads"] // h
    at = torch.arange(longest, device="cuda")
    slots = s["slots"][(s["offsets"][:-1, None] + at).clamp(max=s["slots"].numel() - 1)]
    keys = _rows(case, s["pool"])[0][slots // case["page"], slots % case["page"]].float()  # [request, token, head, dim]
    # Each request's queries, padded to the most that one has.
    first = torch.searchsorted(s["requests"], torch.arange(r + 1, dtype=torch.int32, device="cuda"))
    number = first[:-1, None] + torch.arange(most, device="cuda")
    ends = torch.where(number < first[1:, None], s["ends"][number.clamp(max=len(s["requests"]) - 1)], 0)
    queries = s["queries"][number.clamp(max=len(s["requests"]) - 1)].float() * d ** -0.5
    queries = queries.view(r, most, h, g, d).permute(0, 2, 1, 3, 4).reshape(r, h, most * g, d)
    live = (at < ends[:, :, None]).repeat_interleave(g, dim=1)[:, None]  # [request, 1, query and head, token]
    scores = torch.matmul(queries, keys.permute(0, 2, 3, 1).contiguous()).masked_fill_(~live, -math.inf)
    weights = torch.exp(scores - scores.amax(dim=3, keepdim=True).clamp(min=-3e38)).masked_fill_(~live, 0.0)
    weights /= weights.sum(dim=3, keepdim=True).clamp(min=1e-37)
    sums = weights.sum(dim=2)  # [request, head, token]
    position = torch.arange(s["weights"].shape[1], device="cuda")
    owner = torch.searchsorted(s["offsets"], position, right=True) - 1
    s["weights"] += sums[owner, :, position - s["offsets"][owner]].t()
    return s["weights"]


def _plain_evict(case, s):
    r, h, page = case["requests"], case["heads"], case["page"]
    at = torch.arange(s["longest"], device="cuda")
    number = (s["offsets"][:-1, None] + at).clamp(max=s["tokens"] - 1)
    weights = s["weights"][:, number].transpose(0, 1)  # [request, head, token]
    first, last = _forced_tokens(case).values()
    lengths = s["lengths"][:, None, None]
    rank = torch.where((at < first) | (at >= lengths - last), 0, 1)
    rank = torch.where(at < lengths, rank, 2).expand_as(weights)
    s["kept"].copy_(_best(weights, rank, case["keep"]))
    # Destination position by destination position (request, then place in its list).
    position = torch.arange(s["to_tokens"], device="cuda")
    owner = torch.searchsorted(s["to_offsets"], position, right=True) - 1
    source = s["kept"][owner, :, position - s["to_offsets"][owner]].long() + s["offsets"][owner][:, None]  # [position, head]
    heads = torch.arange(h, device="cuda")
    slots, to_slots = s["slots"][source], s["to_slots"][:, None]
    for to, rows in zip(_rows(case, s["to_pool"]), _rows(case, s["pool"])):
        to[to_slots // page, to_slots % page, heads] = rows[slots // page, slots % page, heads]
    s["to_weights"].copy_(torch.gather(s["weights"], 1, source.t()))
    return [s["kept"], s["to_pool"], s["to_weights"]]


_PLAIN = dict(bounds=_plain_bounds, select=_plain_select, attend=_plain_attend, weights=_plain_weights, evict=_plain_evict)


def run(state):
    case = state["case"]
    return _run_own(case, state) if own else _PLAIN[case["op"]](case, state)


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    op, h, d, page = case["op"], case["heads"], case["dim"], case["page"]
    if op == "bounds":
        tokens = case["pages"] * (page if case["full"] else (page + 1) / 2)
        return dict(bytes=2 * h * d * (tokens + 2 * case["pages"]), flops=0)
    if op == "evict":
        lengths = _ragged(case["requests"], case["low"], case["high"])
        kept = sum(min(n, case["keep"]) for n in lengths)
        return dict(bytes=4 * h * sum(lengths) + kept * h * (2 * 4 * d + 2 * 4 + 4), flops=0)
    lengths, counts = _counts(case)
    queries = sum(counts)
    rows = 2 * case["qheads"] * d * queries
    ends = np.concatenate([n - c + 1 + np.arange(c) for n, c in zip(lengths, counts)])
    if op == "weights":
        return dict(bytes=rows + (2 * d + 8) * h * sum(lengths), flops=2.0 * case["qheads"] * d * int(ends.sum()))
    pages = -(-ends // page)
    listed_pages = np.minimum(pages, case["keep"])
    if op == "select":
        return dict(bytes=rows + 4 * h * (d * sum(-(-n // page) for n in lengths) + int(listed_pages.sum())),
                    flops=2.0 * case["qheads"] * d * int(pages.sum()))
    # What the queries of a request list, at most its own tokens.
    tokens = listed_pages * page - (pages * page - ends)
    rows_read = np.minimum(np.add.reduceat(tokens, np.cumsum([0] + counts[:-1])), lengths)
    tokens = int(tokens.sum())
    return dict(bytes=2 * rows + h * (4 * d * int(rows_read.sum()) + 4 * int(listed_pages.sum())),
                flops=4.0 * case["qheads"] * d * tokens)


# ---- the definitions in 64 bits -------------------------------------------------------------


def exact(case, seed):
    """What run() returns, sequence by sequence and in 64 bits."""
    s = _PREPARE[case["op"]](case, _generator(seed))
    return _EXACT[case["op"]](case, s)


def _layer_tokens(case, pool, tensor):
    """[slot, head, dim] of the layer's keys (0) or values (1)."""
    rows = pool[:, _LAYER, tensor]
    h, d, page = case["heads"], case["dim"], case["page"]
    if case["hnd"]:
        rows = rows.reshape(-1, h, page, d).permute(0, 2, 1, 3)
    return rows.reshape(-1, h, d)


def _exact_bounds(case, s):
    keys = _layer_tokens(case, s["pool"], 0).view(-1, case["page"], case["heads"], case["dim"])
    bounds = s["bounds"].double()
    by_count = {}
    for page, count in zip(s["pages"].tolist(), s["counts"].tolist()):
        by_count.setdefault(count, []).append(page)
    for count, pages in by_count.items():
        at = torch.tensor(pages, device="cuda")
        bounds[at] = torch.stack(torch.aminmax(keys[at, :count].double(), dim=1), dim=2)
    return bounds


def _ranked(order, forced, keep):
    """The first `keep` of the forced ones and then of `order`, ascending, filled up with -1."""
    rest = order[~np.isin(order, forced)]
    chosen = np.sort(np.concatenate([forced, rest])[:keep])
    return np.concatenate([chosen, np.full(keep - len(chosen), -1, np.int64)])


def _exact_select(case, s):
    page, h, d, keep = case["page"], case["heads"], case["dim"], case["keep"]
    first, last = (min(v, keep // 2) for v in _FORCED.values())
    chosen = []
    for q, (request, end) in enumerate(zip(s["requests"].tolist(), s["ends"].tolist())):
        count = -(-end // page)
        begin = int(s["offsets"][request])
        bounds = s["bounds"][s["slots"][begin:begin + end:page] // page].double()
        scores = torch.full((h, count), -math.inf, dtype=torch.float64, device="cuda")
        for i in range(case["qheads"] // h):
            vector = s["queries"][q].view(h, -1, d)[:, i].double()[None, :, None]
            scores = torch.maximum(scores, (vector * bounds).amax(dim=2).sum(dim=2).t())
        forced = np.unique(np.concatenate([np.arange(min(first, count)), np.arange(max(0, count - last), count)]))
        order = np.argsort(-scores.cpu().numpy(), axis=1, kind="stable")
        chosen.append(np.stack([_ranked(order[k], forced, keep) for k in range(h)]))
    return torch.from_numpy(np.stack(chosen).astype(np.int32))


def _exact_attend(case, s):
    page, h, d = case["page"], case["heads"], case["dim"]
    keys, values = (_layer_tokens(case, s["pool"], t) for t in (0, 1))
    output = torch.zeros(s["output"].shape, dtype=torch.float64, device="cuda")
    group = case["qheads"] // h
    for q, (request, end) in enumerate(zip(s["requests"].tolist(), s["ends"].tolist())):
        slots = s["slots"][int(s["offsets"][request]):][:end]
        listed_pages = s["selected"][q].cpu().numpy()
        for k in range(h):
            token = (listed_pages[k][listed_pages[k] >= 0][:, None] * page + np.arange(page)).reshape(-1)
            at = slots[torch.from_numpy(token[token < end]).to("cuda")]
            mine = s["queries"][q, k * group:(k + 1) * group].double()
            weights = torch.softmax(mine @ keys[at, k].double().t().contiguous() * d ** -0.5, dim=1)
            output[q, k * group:(k + 1) * group] = weights @ values[at, k].double()
    return output


def _exact_weights(case, s):
    h, d = case["heads"], case["dim"]
    keys = _layer_tokens(case, s["pool"], 0)
    total = s["weights"].double()
    first = 0
    for request, (length, count) in enumerate(zip(s["lengths"], s["counts"])):
        begin = int(s["offsets"][request])
        mine = keys[s["slots"][begin:begin + length]].double()
        dead = torch.arange(length, device="cuda")[None, None, :] >= s["ends"][first:first + count, None, None]
        for k in range(h):
            queries = s["queries"][first:first + count].view(count, h, -1, d)[:, k].double()
            scores = (queries.reshape(-1, d) @ mine[:, k].t().contiguous()).view(count, -1, length) * d ** -0.5
            total[k, begin:begin + length] += torch.softmax(scores.masked_fill_(dead, -math.inf), dim=2).sum(dim=(0, 1))
        first += count
    return total


def _exact_evict(case, s):
    h, keep = case["heads"], case["keep"]
    first, last = _forced_tokens(case).values()
    weights, slots, offsets = s["weights"].double().cpu().numpy(), s["slots"].cpu().numpy(), s["offsets"].tolist()
    kept, sources = [], []
    for request, length in enumerate(s["lengths"].tolist()):
        begin = offsets[request]
        forced = np.unique(np.concatenate([np.arange(min(first, length)), np.arange(max(0, length - last), length)]))
        order = np.argsort(-weights[:, begin:begin + length], axis=1, kind="stable")
        kept.append(np.stack([_ranked(order[k], forced, keep) for k in range(h)]))
        sources.append(kept[-1][:, :min(length, keep)] + begin)
    source = np.concatenate(sources, axis=1)  # [head, destination position]
    to_slots = s["to_slots"]
    out = s["to_pool"].clone()
    for tensor in (0, 1):
        rows = _layer_tokens(case, s["pool"], tensor)
        to = torch.zeros(out.shape[0] * case["page"], h, case["dim"], dtype=torch.bfloat16, device="cuda")
        for k in range(h):
            to[to_slots, k] = rows[torch.from_numpy(slots[source[k]]).to("cuda"), k]
        to = to.view(-1, case["page"], h, case["dim"])
        out[:, _LAYER, tensor] = (to.transpose(1, 2) if case["hnd"] else to).reshape(out.shape[0], -1)
    moved = np.take_along_axis(weights, source, axis=1)
    return [torch.from_numpy(np.stack(kept).astype(np.int32)), out.double(), torch.from_numpy(moved)]


_EXACT = dict(bounds=_exact_bounds, select=_exact_select, attend=_exact_attend, weights=_exact_weights,
              evict=_exact_evict)
