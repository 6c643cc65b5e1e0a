"""Cases that measure the key/value cache operators of generation: ``zoo.ops.paged_append``,
``zoo.ops.paged_attention`` and ``zoo.ops.paged_evict``.

A cache is a pool of pages ``[pages, kv_heads, page, dim]`` for the keys and one for the values. Row b of
``page_table`` names the pages of sequence b in order, so slot s of sequence b is page ``page_table[b, s // page]``,
row ``s % page``. ``lengths[b]`` slots are in use. Where eviction is on, two more pools of the shape
``[pages, kv_heads, page]`` hold the attention weight each slot has gathered and the position of its token; every
kv head may hold other tokens of the sequence than its neighbour, so both have a head axis.

``own = False`` computes the operators from elementary torch operations.
"""
import math
import os
import sys

import torch

own = False
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "analytics-zoo_amd"))

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one sentence of the default TransformerLayer (12 heads of 64, 77 positions): launch latency
        {"name": "attend one sentence", "op": "attend", "dtype": "bf16", "batch": 1, "heads": 12, "kv_heads": 12,
         "dim": 64, "page": 16, "longest": 77, "ragged": False, "weights": False},
        # a serving batch at BERT-base's head layout, 512 positions, weights gathered for eviction
        {"name": "attend batch, weights", "op": "attend", "dtype": "bf16", "batch": 32, "heads": 12, "kv_heads": 12,
         "dim": 64, "page": 64, "longest": 512, "ragged": True, "weights": True},
        # grouped heads, lengths from an idle row to 8k, half precision
        {"name": "attend grouped, ragged", "op": "attend", "dtype": "fp16", "batch": 24, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "longest": 8192, "ragged": True, "weights": False},
        # the cache in 32 bits, a head width and a page size that fit no tile
        {"name": "attend fp32, odd sizes", "op": "attend", "dtype": "fp32", "batch": 5, "heads": 21, "kv_heads": 7,
         "dim": 80, "page": 24, "longest": 2999, "ragged": True, "weights": True},
        # one long document: the length has to be split to fill the chip
        {"name": "attend one long document", "op": "attend", "dtype": "bf16", "batch": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 128, "longest": 131072, "ragged": False, "weights": True},
        # the largest: a full batch of long sequences
        {"name": "attend full batch", "op": "attend", "dtype": "bf16", "batch": 64, "heads": 64, "kv_heads": 8,
         "dim": 128, "page": 64, "longest": 16384, "ragged": False, "weights": False},
        # the token of a decoding step, at the serving batch's layout
        {"name": "append tokens", "op": "append", "dtype": "bf16", "batch": 32, "heads": 12, "kv_heads": 12, "dim": 64,
         "page": 64, "longest": 512, "ragged": True, "tokens": 1},
        # prompts of unequal length in one padded batch
        {"name": "append prompts", "op": "append", "dtype": "bf16", "batch": 16, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "longest": 1000, "ragged": True, "tokens": 2048},
        # one token over the budget: the steady state of a decoding step
        {"name": "evict one", "op": "evict", "dtype": "bf16", "batch": 32, "heads": 12, "kv_heads": 12, "dim": 64,
         "page": 64, "longest": 513, "ragged": False, "budget": 512, "recent": 128},
        # prompts cut down to a quarter before decoding starts
        {"name": "evict prompts", "op": "evict", "dtype": "bf16", "batch": 32, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "longest": 8192, "ragged": True, "budget": 2048, "recent": 256},
        # one long document cut down
        {"name": "evict one long document", "op": "evict", "dtype": "bf16", "batch": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 128, "longest": 131072, "ragged": False, "budget": 16384, "recent": 1024},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "evict"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    kv = rng.choice([1, 2, 4, 7, 8, 12, 16])
    group = rng.choice([1, 1, 2, 3, 4, 8, 16, 24])
    dim = rng.choice([16, 40, 64, 64, 80, 96, 128, 128, 128, 200, 256])
    page = rng.choice([1, 7, 16, 16, 24, 32, 64, 64, 100, 128, 256])
    batch = _log(rng, 1, 96)
    # a quarter of the largest case's keys and values at most, and no more than 8M (head, slot) pairs
    most = min(2 ** 28 // (dim * SIZE[dtype]), 2 ** 21) // (batch * kv)
    longest = _log(rng, 1, max(1, min(131072, most)))
    case = {"op": op, "dtype": dtype, "batch": batch, "heads": kv * group, "kv_heads": kv, "dim": dim, "page": page,
            "longest": longest, "ragged": rng.random() < 0.7}
    if op == "attend":
        case["weights"] = rng.random() < 0.5
    elif op == "append":
        case["tokens"] = rng.choice([1, _log(rng, 1, max(1, min(4096, most * 2 // (group + 2))))])
    else:
        case["budget"] = _log(rng, 1, max(1, longest))
        case["recent"] = rng.randint(0, case["budget"])
    return case


def _lengths(case):
    """The lengths of a case's sequences, the same for every seed up to their order."""
    n, longest = case["batch"], case["longest"]
    if not case["ragged"]:
        return [longest] * n
    got = [max(1, -(-longest * (i + 1) // n)) for i in range(n)]
    if n >= 4:
        got[0] = 0          # an idle row of the serving batch
    return got


def _counts(case):
    """Tokens that each sequence of an append case brings."""
    n, t = case["batch"], case["tokens"]
    return [max(1, -(-t * (n - i) // n)) if case["ragged"] else t for i in range(n)]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    host = torch.Generator()
    host.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    B, Hq, H, D, page = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    order = torch.randperm(B, generator=host)
    lengths = torch.tensor(_lengths(case), dtype=torch.int32)[order]
    counts = torch.tensor(_counts(case), dtype=torch.int32)[order] if case["op"] == "append" else None
    need = lengths if counts is None else lengths + counts
    owned = (need + page - 1) // page
    width = max(1, int(owned.max()))
    total = int(owned.sum())
    pages = total + total // 16 + 1         # some pages belong to nobody in this batch
    ids = torch.randperm(pages, generator=host)[:total].int()
    table = torch.full((B, width), -1, dtype=torch.int32)
    table[torch.arange(width)[None, :] < owned[:, None]] = ids
    s = {"op": case["op"], "lengths": lengths.to(dev), "table": table.to(dev)}
    s["k"] = torch.randn(pages, H, page, D, generator=gen, device=dev, dtype=dt)
    s["v"] = torch.randn(pages, H, page, D, generator=gen, device=dev, dtype=dt)
    if case["op"] == "attend":
        # keys and queries of trained models meet in logits a few units wide
        s["q"] = torch.randn(B, Hq, D, generator=gen, device=dev, dtype=dt) * 2
        s["scores"] = None
        if case["weights"]:
            s["scores"] = torch.rand(pages, H, page, generator=gen, device=dev)
            s["scores_out"] = torch.zeros_like(s["scores"])
        return s
    s["scores"] = torch.rand(pages, H, page, generator=gen, device=dev)
    if case["op"] == "append":
        # the projection's output, queries, keys and values of a token side by side
        s["qkv"] = torch.randn(B, case["tokens"], Hq + 2 * H, D, generator=gen, device=dev, dtype=dt)
        s["split"] = (Hq, H)
        s["counts"] = counts.to(dev)
        s["positions"] = torch.zeros(pages, H, page, dtype=torch.int32, device=dev)
        s["seen"] = s["lengths"] + 11       # tokens that eviction has taken before
        return s
    # gathered weight falls off over a few orders of magnitude; a slot in sixteen was never looked at
    s["scores"] = torch.exp(torch.randn(pages, H, page, generator=gen, device=dev) * 2 - 4)
    s["scores"] *= (torch.rand(pages, H, page, generator=gen, device=dev) > 1 / 16).float()
    # positions of the slots: a shuffle of the tokens seen, another one for each head
    slot, ok, pg, off = _slots(s["table"], s["lengths"], page)
    mix = torch.rand(B, H, slot.numel(), generator=gen, device=dev) + (~ok)[:, None, :] * 2.0
    rank = mix.argsort(-1).argsort(-1).int()
    s["positions"] = torch.zeros(pages, H, page, dtype=torch.int32, device=dev)
    b, n = ok.nonzero(as_tuple=True)
    s["positions"][pg[b, n], :, off[n]] = rank[b, :, n] + 5
    s["seen"] = s["lengths"] + 5
    s["scores_out"] = torch.zeros_like(s["scores"])
    s["positions_out"] = torch.zeros_like(s["positions"])
    s["budget"], s["recent"] = case["budget"], case["recent"]
    return s


def _slots(table, lengths, page):
    """(slot numbers [S], slots in use [B, S], their pages [B, S], their rows in the page [S])."""
    slot = torch.arange(table.shape[1] * page, device=table.device)
    ok = slot[None, :] < lengths[:, None]
    return slot, ok, table[:, slot // page].clamp(min=0).long(), slot % page


def _attend(q, k, v, table, lengths, scores, scores_out):
    B, Hq, D = q.shape
    H, page = k.shape[1], k.shape[2]
    slot, ok, pg, off = _slots(table, lengths, page)
    S = slot.numel()
    t = table.clamp(min=0).long()
    keys = k[t].transpose(1, 2).reshape(B, H, S, D).float()
    w = torch.matmul(q.float().view(B, H, Hq // H, D), keys.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    del keys
    w = w.masked_fill(~ok[:, None, None, :], float("-inf"))
    w = torch.exp(w - w.amax(-1, keepdim=True).clamp(min=-3e38))
    w = w / w.sum(-1, keepdim=True).clamp(min=1e-38)
    values = v[t].transpose(1, 2).reshape(B, H, S, D).float()
    values = values.masked_fill(~ok[:, None, :, None], 0.0)
    o = torch.matmul(w, values).view(B, Hq, D).to(q.dtype)
    if scores is None:
        return o
    b, n = ok.nonzero(as_tuple=True)
    at = (pg[b, n], slice(None), off[n])
    scores_out[at] = scores[at] + w.sum(2)[b, :, n]
    return o, scores_out


def _append(k, v, k_pages, v_pages, table, lengths, counts, seen, scores, positions):
    page = k_pages.shape[2]
    t = torch.arange(k.shape[1], device=k.device)
    b, n = (t[None, :] < counts[:, None]).nonzero(as_tuple=True)
    slot = lengths[b] + n
    at = (table[b, slot // page].long(), slice(None), (slot % page).long())
    k_pages[at] = k[b, n]
    v_pages[at] = v[b, n]
    scores[at] = 0.0
    positions[at] = (seen[b] + n).int()[:, None]
    return k_pages, v_pages, scores, positions, lengths + counts


def _evict(k, v, scores, positions, table, lengths, seen, budget, recent, scores_out, positions_out):
    B, H, page = table.shape[0], k.shape[1], k.shape[2]
    slot, ok, pg, off = _slots(table, lengths, page)
    S = slot.numel()
    score = scores[pg, :, off].transpose(1, 2)          # [B, H, S]
    pos = positions[pg, :, off].transpose(1, 2)
    late = pos >= (seen - recent)[:, None, None]
    key = score.masked_fill(late, float("inf")).masked_fill(~ok[:, None, :], float("-inf"))
    rank = torch.empty_like(key, dtype=torch.int64)
    rank.scatter_(-1, key.sort(dim=-1, descending=True, stable=True)[1], slot.expand(B, H, S))
    kept = (rank < budget) & ok[:, None, :]
    hole = ~kept & ok[:, None, :] & (slot < budget)
    tail = kept & (slot >= budget)
    # the i-th hole, in slot order, takes the i-th kept slot behind the budget
    nth = tail.cumsum(-1) - 1
    source = torch.zeros(B, H, S + 1, dtype=torch.int64, device=k.device)
    source.scatter_(-1, torch.where(tail, nth, S), slot.expand(B, H, S))
    b, h, d = (kept & (slot < budget)).nonzero(as_tuple=True)
    scores_out[pg[b, d], h, off[d]] = scores[pg[b, d], h, off[d]]
    positions_out[pg[b, d], h, off[d]] = positions[pg[b, d], h, off[d]]
    b, h, d = hole.nonzero(as_tuple=True)
    src = source[b, h, (hole.cumsum(-1) - 1)[b, h, d]]
    to, fr = (pg[b, d], h, off[d]), (pg[b, src], h, off[src])
    k[to] = k[fr]
    v[to] = v[fr]
    scores_out[to] = scores[fr]
    positions_out[to] = positions[fr]
    return k, v, scores_out, positions_out, lengths.clamp(max=budget)


def run(s):
    k, v, table, lengths = s["k"], s["v"], s["table"], s["lengths"]
    if own:
        from zoo import ops
    if s["op"] == "attend":
        if not own:
            return _attend(s["q"], k, v, table, lengths, s["scores"], s.get("scores_out"))
        o = ops.paged_attention(s["q"], k, v, table, lengths, scores=s["scores"], scores_out=s.get("scores_out"))
        return o if s["scores"] is None else (o, s["scores_out"])
    if s["op"] == "append":
        hq, h = s["split"]
        new_k, new_v = s["qkv"][:, :, hq:hq + h], s["qkv"][:, :, hq + h:]
        if not own:
            return _append(new_k, new_v, k, v, table, lengths, s["counts"], s["seen"], s["scores"], s["positions"])
        n = ops.paged_append(new_k, new_v, k, v, table, lengths, counts=s["counts"], seen=s["seen"],
                                scores=s["scores"], positions=s["positions"])
        return k, v, s["scores"], s["positions"], n
    if not own:
        return _evict(k, v, s["scores"], s["positions"], table, lengths, s["seen"], s["budget"], s["recent"],
                      s["scores_out"], s["positions_out"])
    n = ops.paged_evict(k, v, s["scores"], s["positions"], table, lengths, s["seen"], s["budget"], s["recent"],
                           scores_out=s["scores_out"], positions_out=s["positions_out"])
    return k, v, s["scores_out"], s["positions_out"], n


def work(case):
    size, H, D, page = SIZE[case["dtype"]], case["kv_heads"], case["dim"], case["page"]
    lens = _lengths(case)
    total = sum(lens)
    if case["op"] == "attend":
        b = 2 * total * H * D * size + 2 * case["batch"] * case["heads"] * D * size
        b += 4 * sum(-(-n // page) for n in lens) + 4 * len(lens)
        if case["weights"]:
            b += 8 * total * H              # gathered weight read and written
        return {"bytes": b, "flops": 4 * total * case["heads"] * D}
    if case["op"] == "append":
        n = sum(_counts(case))
        return {"bytes": n * H * (4 * D * size + 8) + 16 * len(lens), "flops": 0}
    # Weights and positions of every slot read, those of the kept ones written, and the rows that move: a kept
    # slot behind the budget for each evicted one before it. The kept share of the slots that are not recent:
    b = 16 * len(lens)
    for n in lens:
        K, R = case["budget"], case["recent"]
        if n > K:
            moved = (n - K) * (K / n)       # positions are shuffled, so a slot is kept with K / n wherever it lies
            b += H * (8 * n + 8 * K + moved * 4 * D * size)
        else:
            b += H * 16 * n
    return {"bytes": b, "flops": 0}


def exact(case, seed):
    """Attention in 64 bits, sequence by sequence; what is appended or moved is no computed number."""
    if case["op"] != "attend":
        return None
    s = prepare(case, seed)
    B, Hq, H, D, page = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    o = torch.zeros(B, Hq, D, dtype=torch.float64, device="cuda")
    total = s["scores_out"].double() if case["weights"] else None
    for b in range(B):
        n = int(s["lengths"][b])
        if n == 0:
            continue
        ids = s["table"][b, :-(-n // page)].long()
        at = torch.arange(n, device="cuda")
        for h in range(H):
            rows = s["k"][ids, h].reshape(-1, D)[:n].double()
            vals = s["v"][ids, h].reshape(-1, D)[:n].double()
            qh = s["q"].double()[b].reshape(H, Hq // H, D)[h]
            w = torch.softmax((qh @ rows.T) / math.sqrt(D), -1)
            o[b].view(H, Hq // H, D)[h] = w @ vals
            if total is not None:
                pg = ids[at // page]
                total[pg, h, at % page] = s["scores"].double()[pg, h, at % page] + w.sum(0)
    return o if total is None else (o, total)
