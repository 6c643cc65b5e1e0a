"""The key/value cache of token-by-token generation with a causal TransformerLayer.

Keys and values lie in two pools of pages, ``k_pages`` and ``v_pages`` ``[pages, kv_heads, page, dim]``;
``page_table`` (int32 ``[batch, width]``) names the pages of each sequence in order: slot ``s`` of
sequence ``b`` is row ``s % page`` of page ``page_table[b, s // page]``. ``lengths`` (int32 ``[batch]``)
says how many slots are in use. Entries of the table behind the last slot in use are never read.

    paged_append      writes the keys and values of new tokens behind the slots in use
    paged_attention   attention of one new token per sequence over the slots in use
    paged_evict       cuts sequences down to a budget of slots, by the attention weight each slot gathered

Eviction needs two more pools ``[pages, kv_heads, page]``: ``scores`` (float32, the attention weight a slot
has gathered) and ``positions`` (int32, which token a slot holds). Both have a head axis, because after an
eviction each kv head may hold other tokens.

Lengths and tables are read on the device only, so a decoding step can be captured into a hipGraph. What
cannot be checked on the host is never followed: a length below 0 or past the table (or ``max_length``), or
a page id outside the pools, makes the attention of that sequence NaN; its tokens on such pages are not
written, and it is not evicted from. A page that is written (by ``paged_append``, ``paged_evict`` or as
``scores_out``) must belong to one row of the table only, and once; pages that are only read may be
shared.

On the GPU these run on the kernels of csrc/kernels/kvcache.hip for bfloat16, float16 and float32 caches with
a head dimension that is a multiple of 8 up to 256 and at most 256 query heads to a kv head; K/V rows may be
strided in any order as long as each row is contiguous and starts on 16 bytes. CPU tensors run on the
PyTorch implementation below. There is no backward pass: inputs that require gradients are refused.

Extends TransformerLayer (Zs/pipeline/api/keras/layers/TransformerLayer.scala:137-181), which the
reference only evaluates over whole sequences.
"""
import math

import torch

from zoo.ops._native import native


def _no_grad(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("%s has no backward pass: call it under torch.no_grad()" % what)


def paged_attention(q, k_pages, v_pages, page_table, lengths, scale=None, scores=None, scores_out=None,
                    max_length=None):
    """Attention of one token per sequence: ``q`` [batch, heads, dim] over the first ``lengths[b]`` slots, the
    heads of ``q`` in equal consecutive groups per kv head. Returns [batch, heads, dim], zeros for an empty
    sequence. ``scale`` defaults to 1 / sqrt(dim).

    With ``scores``, every slot in use gathers the weight that the query heads of its kv head gave it:
    ``scores_out[slot] = scores[slot] + sum(weights)``; ``scores_out`` defaults to ``scores`` itself. This takes
    ``batch * heads * capacity`` floats of workspace, where the capacity is what a row of the table can name, or
    ``max_length`` if that is given: no sequence is longer."""
    _no_grad("paged_attention", q, k_pages, v_pages, scores)
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if k_pages.is_cuda:
        return native().paged_attention(q, k_pages, v_pages, page_table, lengths, scale, scores, scores_out, max_length)
    return _attention_ref(q, k_pages, v_pages, page_table, lengths, scale, scores, scores_out, max_length)


def paged_append(k, v, k_pages, v_pages, page_table, lengths, counts=None, seen=None, scores=None, positions=None):
    """Writes ``k`` / ``v`` [batch, tokens, kv_heads, dim] (strided views of a packed projection will do) into the
    slots from ``lengths[b]`` on. ``counts`` (int32 [batch]): how many tokens of each row are real, for padded
    prompts; all by default. The new slots' ``scores``, if given, become 0 and their ``positions``, if given,
    ``seen[b] + t`` (``seen``: int32 [batch], the tokens each sequence has had; ``lengths`` by default). Returns the
    new lengths as a new tensor. Tokens that the table has no room for are not written, but counted: the
    sequence is then longer than its table and its attention NaN."""
    _no_grad("paged_append", k, v, k_pages, v_pages)
    if k_pages.is_cuda:
        return native().paged_append(k, v, k_pages, v_pages, page_table, lengths, counts, seen, scores, positions)
    return _append_ref(k, v, k_pages, v_pages, page_table, lengths, counts, seen, scores, positions)


def paged_evict(k_pages, v_pages, scores, positions, page_table, lengths, seen, budget, recent=0, scores_out=None,
                positions_out=None):
    """Cuts every sequence longer than ``budget`` slots down to it, for each kv head by itself: kept are the slots of
    the last ``recent`` positions (those >= ``seen[b] - recent``) and then those of the largest score; of equal
    ones the lower slot is kept, and a NaN score counts as the lowest. Kept slots below the budget stay where they
    are; the i-th evicted slot there takes over the i-th kept slot behind the budget, keys, values, score and
    position, so no more rows move than have to. Returns the new lengths ``min(lengths, budget)`` as a new tensor.

    Scores and positions of the kept slots go to ``scores_out`` and ``positions_out``, by default where they were."""
    _no_grad("paged_evict", k_pages, v_pages, scores)
    scores_out = scores if scores_out is None else scores_out
    positions_out = positions if positions_out is None else positions_out
    if k_pages.is_cuda:
        return native().paged_evict(k_pages, v_pages, scores, positions, page_table, lengths, seen, budget, recent,
                                    scores_out, positions_out)
    return _evict_ref(k_pages, v_pages, scores, positions, page_table, lengths, seen, budget, recent, scores_out,
                      positions_out)


# ---------------------------------------------------------------------------- PyTorch implementation
def _check(k_pages, v_pages, page_table, lengths, max_length=None):
    """Capacity of a row of the table; raises what the native bindings raise."""
    def need(ok, msg):
        if not ok:
            raise RuntimeError("paged cache: " + msg)
    need(k_pages.dim() == 4 and k_pages.shape == v_pages.shape and k_pages.dtype == v_pages.dtype,
         "k_pages and v_pages must both be [pages, kv_heads, page, dim]")
    need(page_table.dim() == 2 and page_table.dtype == torch.int32, "page_table must be int32 [batch, width]")
    need(lengths.dtype == torch.int32 and tuple(lengths.shape) == (page_table.shape[0],),
         "lengths must be int32 [batch]")
    need(max_length is None or max_length >= 0, "max_length must not be negative")
    cap = page_table.shape[1] * k_pages.shape[2] if k_pages.shape[0] else 0
    return cap if max_length is None else min(cap, max_length)


def _rows(k_pages, page_table, lengths, cap):
    """For each sequence: its pages and rows in slot order, or None where length or table are bad."""
    out = []
    page = k_pages.shape[2]
    for b, n in enumerate(lengths.tolist()):
        if not 0 <= n <= cap:
            out.append(None)
            continue
        s = torch.arange(n)
        p = page_table[b, s // page].long()
        out.append(None if bool(((p < 0) | (p >= k_pages.shape[0])).any()) else (p, s % page))
    return out


def _attention_ref(q, k_pages, v_pages, page_table, lengths, scale, scores, scores_out, max_length):
    cap = _check(k_pages, v_pages, page_table, lengths, max_length)
    B, Hq, D = q.shape
    H = k_pages.shape[1]
    if Hq < H or Hq % H or D != k_pages.shape[3] or B != page_table.shape[0]:
        raise RuntimeError("paged_attention: q must be [batch, heads, dim], heads a multiple of the cache's kv heads")
    if not math.isfinite(scale):
        raise RuntimeError("paged_attention: scale must be finite")
    if scores is None and scores_out is not None:
        raise RuntimeError("paged_attention: scores_out without scores")
    scores_out = scores if scores_out is None else scores_out
    o = torch.zeros(B, Hq, D, dtype=q.dtype)
    for b, at in enumerate(_rows(k_pages, page_table, lengths, cap)):
        if at is None:
            o[b] = float("nan")
            continue
        if at[0].numel() == 0:
            continue
        ct = torch.promote_types(q.dtype, torch.float32)
        k, v = (t[at[0], :, at[1]].to(ct).transpose(0, 1) for t in (k_pages, v_pages))       # [H, n, D]
        w = torch.softmax(torch.matmul(q[b].to(ct).view(H, Hq // H, D), k.transpose(1, 2)) * scale, -1)
        o[b] = torch.matmul(w, v).reshape(Hq, D).to(q.dtype)
        if scores is not None:
            scores_out[at[0], :, at[1]] = scores[at[0], :, at[1]] + w.sum(1).t().to(scores.dtype)
    return o


def _append_ref(k, v, k_pages, v_pages, page_table, lengths, counts, seen, scores, positions):
    cap = _check(k_pages, v_pages, page_table, lengths)
    B, T, H, D = k.shape
    if v.shape != k.shape or (H, D) != (k_pages.shape[1], k_pages.shape[3]) or B != page_table.shape[0] \
            or k.dtype != k_pages.dtype or v.dtype != k_pages.dtype:
        raise RuntimeError("paged_append: k and v must be [batch, tokens, kv_heads, dim] of the cache's type")
    new = lengths.clone()
    page = k_pages.shape[2]
    for b, n in enumerate(lengths.tolist()):
        if not 0 <= n <= cap:
            continue
        c = T if counts is None else max(0, min(T, int(counts[b])))
        new[b] = n + c
        t = torch.arange(min(c, cap - n))
        p = page_table[b, (n + t) // page].long()
        ok = (p >= 0) & (p < k_pages.shape[0])
        t, p, r = t[ok], p[ok], ((n + t) % page)[ok]
        k_pages[p, :, r] = k[b, t]
        v_pages[p, :, r] = v[b, t]
        if scores is not None:
            scores[p, :, r] = 0.0
        if positions is not None:
            first = n if seen is None else int(seen[b])
            positions[p, :, r] = (first + t).int()[:, None].expand(-1, H)
    return new


def _evict_ref(k_pages, v_pages, scores, positions, page_table, lengths, seen, budget, recent, scores_out,
               positions_out):
    cap = _check(k_pages, v_pages, page_table, lengths)
    if budget < 1 or not 0 <= recent <= budget:
        raise RuntimeError("paged_evict: budget must be at least 1 and recent from 0 to the budget")
    new = lengths.clone()
    for b, at in enumerate(_rows(k_pages, page_table, lengths, cap)):
        if at is None or at[0].numel() == 0:
            continue
        p, r = at
        n = p.numel()
        new[b] = min(n, budget)
        score, pos = scores[p, :, r], positions[p, :, r]                  # [n, H]
        for h in range(k_pages.shape[1]):
            s = torch.where(torch.isnan(score[:, h]), torch.tensor(-math.inf), score[:, h]).double()
            # NaN below -inf, recent above +inf: as ranks in a second column
            tier = torch.where(torch.isnan(score[:, h]), 0, 1)
            tier = torch.where(pos[:, h].long() >= int(seen[b]) - recent, 2, tier)
            s = torch.where(tier == 2, torch.zeros_like(s), s)
            order = torch.argsort(s, descending=True, stable=True)
            order = order[torch.argsort(tier[order], descending=True, stable=True)]
            kept = torch.zeros(n, dtype=torch.bool)
            kept[order[:budget]] = True
            src = torch.arange(n)
            hole = (~kept[:budget]).nonzero().flatten()
            src[hole] = (kept[budget:].nonzero().flatten() + budget)
            src = src[:min(n, budget)]
            m = src.numel()
            for pool, out in ((k_pages, k_pages), (v_pages, v_pages), (scores, scores_out), (positions, positions_out)):
                out[p[:m], h, r[:m]] = pool[p[src], h, r[src]]
    return new
