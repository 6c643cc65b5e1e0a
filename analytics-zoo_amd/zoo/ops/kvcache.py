"""The key/value cache of token-by-token generation with a causal TransformerLayer.

Keys and values lie in two pools of pages, ``k_pages`` and ``v_pages`` ``[pages, kv_heads, page, dim]``;
``page_table`` (int32 ``[batch, width]``) names the pages of each sequence in order: slot ``s`` of
sequence ``b`` is row ``s % page`` of page ``page_table[b, s // page]``. ``lengths`` (int32 ``[batch]``)
says how many slots are in use. Entries of the table behind the last slot in use are never read.

    paged_append      writes the keys and values of new tokens behind the slots in use
    paged_attention   attention of one new token per sequence over the slots in use
    paged_evict       cuts sequences down to a budget of slots, by the attention weight each slot gathered
    PagedKVCache      the pools of all layers of a model and the book of their pages

Eviction needs two more pools ``[pages, kv_heads, page]``: ``scores`` (float32, the attention weight a slot
has gathered) and ``positions`` (int32, which token a slot holds). Both have a head axis, because after an
eviction each kv head may hold other tokens.

Lengths and tables are read on the device only, so a decoding step can be captured into a hipGraph. What
cannot be checked on the host is never followed: a length below 0 or past the table (or ``max_length``), or
a page id outside the pools, makes the attention of that sequence NaN, and its slots gather no weight; its
tokens on such pages are not written, and it is not evicted from. A page that is written (by ``paged_append``, ``paged_evict`` or as
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
import operator

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
    ``batch * heads * capacity`` floats of workspace, where the capacity is what a row of the table can name: pass a
    narrower view of a wide table, or ``max_length``, a bound on the lengths (a sequence that is longer comes out
    NaN)."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if k_pages.is_cuda:
        return native().paged_attention(q, k_pages, v_pages, page_table, lengths, scale, scores, scores_out, max_length)
    _no_grad("paged_attention", q, k_pages, v_pages, scores, scores_out)
    return _attention_ref(q, k_pages, v_pages, page_table, lengths, scale, scores, scores_out, max_length)


def paged_append(k, v, k_pages, v_pages, page_table, lengths, counts=None, seen=None, scores=None, positions=None):
    """Writes ``k`` / ``v`` [batch, tokens, kv_heads, dim] (strided views of a packed projection will do) into the
    slots from ``lengths[b]`` on. ``counts`` (int32 [batch]): how many tokens of each row are real, for padded
    prompts; all by default. The new slots' ``scores``, if given, become 0 and their ``positions``, if given,
    ``seen[b] + t`` (``seen``: int32 [batch], the tokens each sequence has had; ``lengths`` by default). Returns the
    new lengths as a new tensor. Tokens that the table has no room for are not written, but counted: the
    sequence is then longer than its table and its attention NaN."""
    if k_pages.is_cuda:
        return native().paged_append(k, v, k_pages, v_pages, page_table, lengths, counts, seen, scores, positions)
    _no_grad("paged_append", k, v, k_pages, v_pages, scores)
    return _append_ref(k, v, k_pages, v_pages, page_table, lengths, counts, seen, scores, positions)


def paged_evict(k_pages, v_pages, scores, positions, page_table, lengths, seen, budget, recent=0, scores_out=None,
                positions_out=None, slack=0):
    """Cuts every sequence longer than ``budget + slack`` slots down to ``budget``, for each kv head by itself: kept are the slots of
    the last ``recent`` positions (those >= ``seen[b] - recent``) and then those of the largest score; of equal
    ones the lower slot is kept, and a NaN score counts as the lowest. Kept slots below the budget stay where they
    are; the i-th evicted slot there takes over the i-th kept slot behind the budget, keys, values, score and
    position, so no more rows move than have to. A sequence of up to ``budget + slack`` slots keeps them all. Returns the new
    lengths as a new tensor.

    Scores and positions of the kept slots go to ``scores_out`` and ``positions_out``, by default where they were.

    The call takes ``8 * min(budget, capacity - budget)`` bytes of workspace for each sequence and kv head, and for tables
    of more than 16384 slots ``4 * capacity`` and 24 KB more, of which the 24 KB are cleared. The capacity, what a row of the
    table can name, also chooses the form of the kernels: pass a narrower view of a wide table (a sequence that is longer
    than the view keeps all its slots)."""
    scores_out = scores if scores_out is None else scores_out
    positions_out = positions if positions_out is None else positions_out
    if k_pages.is_cuda:
        return native().paged_evict(k_pages, v_pages, scores, positions, page_table, lengths, seen, budget, recent,
                                    scores_out, positions_out, slack)
    _no_grad("paged_evict", k_pages, v_pages, scores, scores_out)
    return _evict_ref(k_pages, v_pages, scores, positions, page_table, lengths, seen, budget, recent, scores_out,
                      positions_out, slack)


def _capturing(t):
    return t.is_cuda and torch.cuda.is_current_stream_capturing()


class PagedKVCache:
    """The caches of all layers of a model that generates for up to ``batch`` sequences at a time, and the host's book
    of their pages. The layers share one page table: layer ``i`` owns the kv heads ``i * kv_heads ..`` of the pools, so
    a page holds the same slots of every layer and one ``paged_evict`` serves them all.

    A row's pages are taken as it grows (:meth:`reserve`) and given back by :meth:`release`; ``pages`` bounds their
    number, by default ``batch`` sequences of ``max_length`` slots. With ``budget``, sequences longer than ``budget +
    slack`` slots are cut down to ``budget`` after a step of theirs; their last ``recent`` tokens stay. ``recent`` is 0 by
    default: give some, or a new token competes with slots that have gathered weight for longer. Weight is gathered by
    :meth:`attend`, so the slots of a prompt start with none, and its first eviction goes by the step before it.

    A step of every layer: :meth:`append`, :meth:`attend` per layer, then :meth:`advance`.

    A captured hipGraph can hold steps of all rows, and takes no pages. So ``reserve`` what a step needs before the capture and before each
    replay (which raises where a replay could not be carried out), and tell the host's book about the replay with
    :meth:`replayed` after it. Between replays rows may be released and filled again. A captured step is laid out for rows
    of ``max_length`` slots, or of all ``pages``: that bounds its workspace, so make it no larger than needed."""

    def __init__(self, n_layer, batch, max_length, kv_heads, head_dim, page=64, pages=None, budget=None, recent=None,
                 slack=0, dtype=None, device=None):
        if min(n_layer, batch, max_length, kv_heads, head_dim, page) < 1:
            raise ValueError("PagedKVCache: sizes must be at least 1")
        if budget is not None and budget < 1:
            raise ValueError("PagedKVCache: budget must be at least 1")
        if slack < 0 or budget is None and (recent is not None or slack):
            raise ValueError("PagedKVCache: recent and slack go with a budget, slack not below 0")
        recent = 0 if recent is None else recent
        if budget is not None and not 0 <= recent <= budget:
            raise ValueError("PagedKVCache: recent must be from 0 to the budget")
        device = torch.device("cuda" if torch.cuda.is_available() else "cpu") if device is None else torch.device(device)
        dtype = (torch.bfloat16 if device.type == "cuda" else torch.float32) if dtype is None else dtype
        self.n_layer, self.kv_heads, self.page, self.max_length = n_layer, kv_heads, page, max_length
        self.budget, self.recent, self.slack = budget, recent, slack
        width = -(-max_length // page)
        pages = batch * width if pages is None else pages
        shape = (pages, n_layer * kv_heads, page)
        self.k = torch.zeros(*shape, head_dim, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.scores = torch.zeros(shape, device=device) if budget is not None else None
        self.positions = torch.zeros(shape, dtype=torch.int32, device=device) if budget is not None else None
        self.page_table = torch.full((batch, width), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)   # slots in use
        self.seen = torch.zeros(batch, dtype=torch.int32, device=device)      # tokens each sequence has had
        self._free = list(range(pages - 1, -1, -1))
        self._pages = [[] for _ in range(batch)]
        self._slots = [0] * batch                                             # the host's copy of lengths

    @property
    def batch(self):
        return len(self._slots)

    def layer(self, i):
        """(k_pages, v_pages, scores, positions) of layer ``i``, views of the pools."""
        h = slice(i * self.kv_heads, (i + 1) * self.kv_heads)
        return (self.k[:, h], self.v[:, h], None if self.scores is None else self.scores[:, h],
                None if self.positions is None else self.positions[:, h])

    def rows(self, rows=None):
        """Row numbers as a list, those from the end as numbers from 0; all of them for None. A row may come once."""
        if rows is None:
            return list(range(self.batch))
        rows = [operator.index(r) for r in rows]
        if not all(-self.batch <= r < self.batch for r in rows):
            raise IndexError("PagedKVCache: rows from 0 to %d" % (self.batch - 1))
        rows = [r % self.batch for r in rows]
        if len(set(rows)) != len(rows):
            raise ValueError("PagedKVCache: a row is named twice")
        return rows

    def not_captured(self, what):
        """Raises where a hipGraph is being captured: ``what`` needs copies from the host, which a replay could not repeat."""
        if _capturing(self.k):
            raise RuntimeError("PagedKVCache: %s cannot be captured" % what)

    @staticmethod
    def _tokens(tokens, rows):
        tokens = [tokens] * len(rows) if isinstance(tokens, int) else [int(t) for t in tokens]
        if len(tokens) != len(rows) or any(t < 0 for t in tokens):
            raise ValueError("PagedKVCache: a number of tokens, not negative, for each row")
        return tokens

    def reserve(self, tokens, rows=None):
        """Takes the pages that ``tokens`` (a number, or one for each row) more tokens of the rows need."""
        rows = self.rows(rows)
        tokens = self._tokens(tokens, rows)
        want = [-(-(self._slots[r] + t) // self.page) for r, t in zip(rows, tokens)]
        if any(self._slots[r] + t > self.max_length for r, t in zip(rows, tokens)):
            raise RuntimeError("PagedKVCache: a sequence would be longer than max_length = %d slots" % self.max_length)
        if sum(max(0, w - len(self._pages[r])) for r, w in zip(rows, want)) > len(self._free):
            raise RuntimeError("PagedKVCache: no pages left")
        if _capturing(self.k) and any(w > len(self._pages[r]) for r, w in zip(rows, want)):
            raise RuntimeError("PagedKVCache: a captured step cannot take pages: reserve() them before the capture")
        for r, w in zip(rows, want):
            n = len(self._pages[r])
            if w > n:
                self._pages[r] += [self._free.pop() for _ in range(w - n)]
                self.page_table[r, n:w] = torch.tensor(self._pages[r][n:], dtype=torch.int32).to(self.page_table.device)

    def release(self, rows=None):
        """Empties rows and gives their pages back."""
        self.not_captured("releasing rows")
        for r in range(self.batch) if rows is None else rows:
            self._free += self._pages[r]
            self._pages[r], self._slots[r] = [], 0
            self.page_table[r] = -1
            self.lengths[r] = 0
            self.seen[r] = 0

    def _table(self):
        # No wider than the pages in hand, which bounds the operators' workspace. A captured step keeps the width it was
        # captured with, so it gets all that a row can come to own.
        width = max(len(own) for own in self._pages)
        if _capturing(self.k):
            width = min(self.page_table.shape[1], self.k.shape[0])
        return self.page_table[:, :max(1, width)]

    def append(self, i, k, v, counts=None, rows=None):
        """``paged_append`` to layer ``i`` of all rows, or of the ``rows`` (int64 [n] on the device, each once); returns the
        new lengths, which :meth:`advance` makes the cache's."""
        kp, vp, scores, positions = self.layer(i)
        at = slice(None) if rows is None else rows
        return paged_append(k, v, kp, vp, self._table()[at], self.lengths[at], counts=counts, seen=self.seen[at],
                            scores=scores, positions=positions)

    def attend(self, i, q, lengths, scale=None, rows=None):
        """``paged_attention`` over layer ``i``, gathering weights if there is a budget."""
        kp, vp, scores, _ = self.layer(i)
        at = slice(None) if rows is None else rows
        return paged_attention(q, kp, vp, self._table()[at], lengths, scale=scale, scores=scores)

    def advance(self, tokens, lengths, rows=None, evict=True):
        """Ends a step that gave the rows ``tokens`` tokens (a number, or one for each row): ``lengths`` are in use now,
        less what eviction takes from these rows."""
        r = self.rows(rows)
        tokens = self._tokens(tokens, r)
        if rows is not None:
            self.not_captured("a step of some rows")
        if rows is None:
            self.seen += lengths - self.lengths
            self.lengths.copy_(lengths)
        else:
            self.seen[r] += lengths - self.lengths[r]
            self.lengths[r] = lengths
        for x, t in zip(r, tokens):
            self._slots[x] += t
        if evict:
            self.evict(rows)

    def _kept_pages(self):
        return min(self.page_table.shape[1], -(-(self.budget + self.slack + 1) // self.page))

    def _cut(self, n):
        return self.budget if n > self.budget + self.slack else n

    def evict(self, rows=None):
        """Cuts the sequences (all, or the ``rows``, a list) that are longer than budget + slack slots down to the
        budget, and gives back the pages that a sequence of budget + slack + 1 slots does not need."""
        r = self.rows(rows)
        if rows is not None:
            self.not_captured("an eviction from some rows")
        if self.budget is None or max((self._slots[x] for x in r), default=0) <= self.budget + self.slack:
            return
        at, keep = slice(None) if rows is None else r, self._kept_pages()
        # a table of the pages that rows own in the steady state: one of all pages would make a captured eviction slow
        table = self.page_table[:, :keep] if _capturing(self.k) else self._table()
        self.lengths[at] = paged_evict(self.k, self.v, self.scores, self.positions, table[at], self.lengths[at],
                                       self.seen[at], self.budget, self.recent, slack=self.slack)
        if _capturing(self.k):      # the eviction leaves rows alone that are longer than its table
            self._slots = [n if n > keep * self.page else self._cut(n) for n in self._slots]
            return
        for x in r:
            self._slots[x] = self._cut(self._slots[x])
        for x in r:
            own = self._pages[x]
            if len(own) > keep:
                self._free += own[keep:]
                del own[keep:]
                self.page_table[x, keep:] = -1

    def replayed(self, tokens=1, evicts=False):
        """Tells the host's book that a captured step, which gave every row ``tokens`` tokens and ended with an eviction
        if ``evicts`` (as it does if a row was past budget + slack when it was captured), was replayed; the capture itself
        has been counted, as the first replay. A capture of several steps counts once for each. A captured eviction leaves
        out rows that are more than a page past budget + slack, such as new prompts: they are cut down here."""
        slots = [n + tokens for n in self._slots]      # in use before the eviction
        if any(n > len(own) * self.page for n, own in zip(slots, self._pages)):
            raise RuntimeError("PagedKVCache: the replayed step ran past the pages that were reserved for it")
        self._slots = slots
        if evicts:
            most = self._kept_pages() * self.page
            self._slots = [n if n > most else self._cut(n) for n in slots]
            if max(slots) > most:
                self.evict([r for r, n in enumerate(slots) if n > most])


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


def _apart(k_pages, v_pages):
    if k_pages.numel() and k_pages.data_ptr() == v_pages.data_ptr():
        raise RuntimeError("paged cache: k_pages and v_pages are the same memory")


def _out(out, pool):
    if out.numel() and out.data_ptr() == pool.data_ptr() and \
            any(n > 1 and x != y for n, x, y in zip(out.shape, out.stride(), pool.stride())):
        raise RuntimeError("paged cache: a pool is written over itself in another layout")


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
    if scores is not None:
        _out(scores_out, scores)
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
    if T >= 2 ** 30:
        raise RuntimeError("paged_append: too many tokens in one call")
    _apart(k_pages, v_pages)
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
               positions_out, slack):
    cap = _check(k_pages, v_pages, page_table, lengths)
    if budget < 1 or not 0 <= recent <= budget:
        raise RuntimeError("paged_evict: budget must be at least 1 and recent from 0 to the budget")
    if slack < 0:
        raise RuntimeError("paged_evict: slack must not be negative")
    _apart(k_pages, v_pages)
    _out(scores_out, scores)
    _out(positions_out, positions)
    new = lengths.clone()
    for b, at in enumerate(_rows(k_pages, page_table, lengths, cap)):
        if at is None or at[0].numel() == 0:
            continue
        p, r = at
        n = p.numel()
        keep = budget if n > budget + slack else max(n, budget)
        new[b] = min(n, keep)
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
            kept[order[:keep]] = True
            src = torch.arange(n)
            hole = (~kept[:keep]).nonzero().flatten()
            src[hole] = (kept[keep:].nonzero().flatten() + keep)
            src = src[:min(n, keep)]
            m = src.numel()
            for pool, out in ((k_pages, k_pages), (v_pages, v_pages), (scores, scores_out), (positions, positions_out)):
                out[p[:m], h, r[:m]] = pool[p[src], h, r[src]]
    return new
