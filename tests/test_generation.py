"""Token-by-token running of a causal TransformerLayer over a paged key/value cache: append, attention, eviction and
the host's book of pages as they are used together."""
import pytest
import torch

from zoo.ops import PagedKVCache, paged_append, paged_attention, paged_evict
from zoo.pipeline.api.keras.layers import TransformerLayer

DEVS = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
VOCAB = 60


def layer(dev, hidden=64, heads=4, blocks=2, std=0.3, seq_len=48):
    torch.manual_seed(3)
    t = TransformerLayer.init(vocab=VOCAB + 200, seq_len=seq_len, n_block=blocks, hidden_size=hidden, n_head=heads,
                              initializer_range=std)
    return t.to(dev).eval()


def ids(B, T, dev, first=0):
    g = torch.Generator().manual_seed(1)
    tok = torch.randint(0, VOCAB, (B, T), generator=g)
    pos = (torch.arange(T) + VOCAB + first).expand(B, T)
    return tok.to(dev), pos.to(dev)


def near(a, b, dev, hidden=64, std=0.3):
    """The outputs of a block's LayerNorm are of size 1. On the CPU both sides are float32. On the GPU either rounds its
    activations to bfloat16 at about ten places per block, 2^-9 rms each (a uniform error of at most 2^-8), and both
    do: sqrt(2 * 10 * blocks) 2^-9 = 0.012 of the norm for 2 blocks. The softmax magnifies that: queries and keys
    have components of size std sqrt(hidden), so logits are of size std^2 hidden (23 for 256 wide and 0.3), a relative
    error e of queries or keys moves a logit by e std^2 hidden, and the weights by as much relative to themselves: an
    error of 0.012 (1 + std^2 hidden), with 2 for the estimate's own spread."""
    a, b = a.float().cpu(), b.float().cpu()
    tol = 1e-4 if dev == "cpu" else 2 * 0.0124 * (1 + std * std * hidden)
    assert torch.isfinite(a).all()
    assert ((a - b).norm() / b.norm()).item() < tol


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("hidden,heads,page,std", [
    (64, 4, 16, 0.3), (128, 2, 7, 0.3), (256, 2, 64, 0.3), (256, 2, 64, 0.02), (256, 4, 16, 0.02)])
def test_decoding_equals_the_whole_sequence(dev, hidden, heads, page, std):
    t = layer(dev, hidden, heads, std=std)
    tok, pos = ids(3, 40, dev)
    with torch.no_grad():
        want = t([tok, pos])[0]
    cache = t.init_cache(3, page=page)
    near(t.prefill([tok[:, :25], pos[:, :25]], cache), want[:, :25], dev, hidden, std)
    for i in range(25, 40):
        near(t.decode([tok[:, i], pos[:, i]], cache), want[:, i], dev, hidden, std)
    assert cache.lengths.tolist() == [40] * 3 and cache.seen.tolist() == [40] * 3


@pytest.mark.parametrize("dev", DEVS)
def test_padded_prompts_and_rows_that_come_and_go(dev):
    t = layer(dev)
    tok, pos = ids(4, 30, dev)
    counts = [30, 1, 17, 0]
    with torch.no_grad():
        want = t([tok, pos])[0]
    cache = t.init_cache(4, page=8, pages=14)
    out = t.prefill([tok, pos], cache, counts=counts)
    for b, c in enumerate(counts):
        if c:
            near(out[b, :c], want[b, :c], dev)
    assert cache.lengths.tolist() == counts
    # the next token of each row: the sequence as if the padding had never been there
    at = torch.tensor(counts, device=dev)
    nxt, npos = (at + 3) % VOCAB, at + VOCAB
    got = t.decode([nxt, npos], cache)
    for b, c in enumerate(counts):
        one = [torch.cat([tok[b, :c], nxt[b:b + 1]])[None], torch.cat([pos[b, :c], npos[b:b + 1]])[None]]
        with torch.no_grad():
            near(got[b], t(one)[0][0, -1], dev)
    # row 2 leaves and another prompt takes its place; the others go on undisturbed
    cache.release([2])
    assert cache.lengths.tolist() == [31, 2, 0, 1]
    tok2, pos2 = ids(1, 12, dev, first=0)
    t.prefill([tok2, pos2], cache, rows=[2])
    assert cache.lengths.tolist() == [31, 2, 12, 1] and cache.seen.tolist() == [31, 2, 12, 1]
    got = t.decode([nxt, npos + 1], cache)
    with torch.no_grad():
        near(got[0], t([torch.cat([tok[0], nxt[:1], nxt[:1]])[None], torch.cat([pos[0], npos[:1], npos[:1] + 1])[None]])[0][0, -1], dev)
        near(got[2], t([torch.cat([tok2[0], nxt[2:3]])[None], torch.cat([pos2[0], npos[2:3] + 1])[None]])[0][0, -1], dev)
    # some rows take a step, the others wait
    before = got
    got = t.decode([nxt[1:3], npos[1:3] + 2], cache, rows=[1, 2])
    assert cache.lengths.tolist() == [32, 4, 14, 2] and cache.seen.tolist() == [32, 4, 14, 2]
    with torch.no_grad():
        near(got[1], t([torch.cat([tok2[0], nxt[2:3], nxt[2:3]])[None],
                        torch.cat([pos2[0], npos[2:3] + 1, npos[2:3] + 2])[None]])[0][0, -1], dev)
    assert torch.isfinite(before.float()).all()
    # the book: no page in two rows
    used = [p for own in cache._pages for p in own]
    assert len(used) == len(set(used)) and not set(used) & set(cache._free) and len(used) + len(cache._free) == 14


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("slack", [0, 5])
def test_eviction_while_decoding(dev, slack):
    """Every head keeps its recent tokens, and its keys and values stay with their positions; a cache
    that never reaches its budget changes nothing."""
    t = layer(dev, blocks=1)
    tok, pos = ids(2, 40, dev)
    free, tight = t.init_cache(2, page=8), t.init_cache(2, page=8, budget=16, recent=6, slack=slack)
    loose = t.init_cache(2, page=8, budget=48)
    for c in (free, tight, loose):
        t.prefill([tok[:, :20], pos[:, :20]], c)
    for i in range(20, 40):
        a, b, _ = (t.decode([tok[:, i], pos[:, i]], c) for c in (free, loose, tight))
        assert torch.equal(a, b)
    n = tight.lengths.tolist()
    assert n[0] == n[1] and 16 <= n[0] <= 16 + slack and tight.seen.tolist() == [40, 40]
    assert len(tight._pages[0]) <= -(-(16 + slack + 1) // 8)
    kf, vf, _, _ = free.layer(0)
    kt, vt, scores, positions = tight.layer(0)
    for b in range(2):
        for h in range(4):
            rows = [(int(tight.page_table[b, s // 8]), s % 8) for s in range(n[b])]
            held = [int(positions[p, h, r]) for p, r in rows]
            assert len(set(held)) == n[b] and set(range(34, 40)) <= set(held)
            for (p, r), x in zip(rows, held):
                q = int(free.page_table[b, x // 8])
                assert torch.equal(kt[p, h, r], kf[q, h, x % 8]) and torch.equal(vt[p, h, r], vf[q, h, x % 8])
    # the weights of a step sum to one for each of the heads
    total = torch.stack([torch.stack([loose.scores[int(loose.page_table[b, s // 8]), :, s % 8] for s in range(40)]).sum(0)
                         for b in range(2)])
    assert torch.allclose(total, torch.full_like(total, 20.0), atol=20 * 40 * 2.0 ** -20)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("hidden,heads", [(64, 4), (128, 2)])
def test_prompts_of_one_token(dev, hidden, heads):
    t = layer(dev, hidden, heads, std=0.02)
    tok, pos = ids(1, 3, dev)
    with torch.no_grad():
        want = t([tok, pos])[0]
    cache = t.init_cache(1, max_length=3, page=1)
    near(t.prefill([tok[:, :1], pos[:, :1]], cache)[:, 0], want[:, 0], dev, hidden, 0.02)
    for i in (1, 2):
        near(t.decode([tok[:, i], pos[:, i]], cache), want[:, i], dev, hidden, 0.02)


def test_refusals():
    t = layer("cpu")
    tok, pos = ids(2, 10, "cpu")
    cache = t.init_cache(2, max_length=12, page=4, pages=5)
    with pytest.raises(RuntimeError, match="no pages left"):
        t.prefill([tok, pos], cache)
    assert cache.lengths.tolist() == [0, 0] and len(cache._free) == 5
    t.prefill([tok, pos], cache, counts=[10, 5])
    with pytest.raises(RuntimeError, match="in use"):
        t.prefill([tok, pos], cache, counts=[1, 1])
    t.decode([tok[:, 0], pos[:, 0]], cache)
    t.decode([tok[:, 0], pos[:, 0]], cache)
    with pytest.raises(RuntimeError, match="max_length"):
        t.decode([tok[:, 0], pos[:, 0]], cache)
    with pytest.raises(ValueError):
        t.decode([tok, pos], cache)
    with pytest.raises(ValueError):
        t.decode([tok[:, 0], pos[:, 0]], cache, rows=[1, 1])
    with pytest.raises(ValueError):
        t.decode([tok[:0, 0], pos[:0, 0]], cache, rows=[])
    with pytest.raises(ValueError):
        t.prefill([tok[:, :0], pos[:, :0]], t.init_cache(2))
    with pytest.raises(ValueError):
        t.prefill([tok, pos], cache, rows=[0])
    with pytest.raises(ValueError):
        t.prefill([tok, pos], t.init_cache(2), counts=[11, 1])
    for bad in (dict(budget=0), dict(budget=4, recent=5), dict(recent=2), dict(slack=1), dict(page=0)):
        with pytest.raises(ValueError):
            t.init_cache(2, **bad)
    t.train()
    with pytest.raises(RuntimeError, match="eval"):
        t.prefill([tok, pos], t.init_cache(2))
    both = TransformerLayer.init(vocab=80, seq_len=8, n_block=1, hidden_size=16, n_head=2, bidirectional=True).eval()
    with pytest.raises(RuntimeError, match="bidirectional"):
        both.prefill([tok % 8, pos % 8], both.init_cache(2, max_length=12))


@pytest.mark.gpu
@pytest.mark.parametrize("budget", [None, 24])
def test_captured_steps(gpu, budget):
    """A captured decoding step, replayed with other work between the replays, does what the eager one does, bit for bit."""
    t = layer("cuda", blocks=2)
    tok, pos = ids(3, 60, "cuda")
    caches = [t.init_cache(3, max_length=80, page=16, budget=budget, recent=8 if budget else None) for _ in range(2)]
    start = 30
    for c in caches:
        t.prefill([tok[:, :start], pos[:, :start]], c)
        t.decode([tok[:, start], pos[:, start]], c)
        c.reserve(30)
    eager, static = caches
    x, p = tok[:, start + 1].clone(), pos[:, start + 1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    spare = t.init_cache(3, max_length=80, page=16, budget=budget)
    with torch.cuda.stream(side):
        t.prefill([tok[:, :4], pos[:, :4]], spare)
        t.decode([x, p], spare)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = t.decode([x, p], static)
    for i in range(start + 1, 55):
        x.copy_(tok[:, i])
        p.copy_(pos[:, i])
        g.replay()
        if i > start + 1:
            static.replayed(1, evicts=budget is not None)
        junk = torch.randn(512, 512, device="cuda") @ torch.randn(512, 512, device="cuda")
        want = t.decode([tok[:, i], pos[:, i]], eager)
        torch.cuda.synchronize()
        assert torch.equal(y, want), i
        assert torch.equal(static.lengths, eager.lengths) and torch.equal(static.seen, eager.seen)
    assert static._slots == eager._slots
    assert torch.isfinite(junk).all()


@pytest.mark.gpu
def test_two_streams_at_once_and_another_stream(gpu):
    """Two sequences of calls on two streams at the same time: each call's workspace is its own."""
    from test_kvcache import make
    args = [make(4, 2, 4, 128, 64, [3000, 700, 0, 2049], torch.bfloat16, "cuda", seed=s) for s in range(2)]
    want = [paged_attention(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged_attention(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


@pytest.mark.gpu
def test_a_step_by_hand(gpu):
    """Append, attend and evict through zoo.ops alone, lengths updated in place, against the CPU implementation."""
    out = {}
    for dev in ("cpu", "cuda"):
        g = torch.Generator().manual_seed(9)
        k, v = (torch.zeros(12, 2, 8, 16).to(dev) for _ in range(2))
        scores, positions = torch.zeros(12, 2, 8).to(dev), torch.zeros(12, 2, 8, dtype=torch.int32).to(dev)
        table = torch.tensor([[3, 1, 7, 5], [0, 11, 2, 9]], dtype=torch.int32).to(dev)
        n = torch.zeros(2, dtype=torch.int32).to(dev)
        seen = n.clone()
        outs = []
        for step in range(40):
            kv = torch.randn(2, 1, 2, 2, 16, generator=g).to(dev)
            q = torch.randn(2, 6, 16, generator=g).to(dev)
            n.copy_(paged_append(kv[:, :, 0], kv[:, :, 1], k, v, table, n, seen=seen, scores=scores, positions=positions))
            seen += 1
            outs.append(paged_attention(q, k, v, table, n, scores=scores).cpu())
            n.copy_(paged_evict(k, v, scores, positions, table, n, seen, 20, 4))
        out[dev] = (torch.stack(outs), positions.cpu(), n.cpu())
    # float32 sums in another order: 2^-24 times a few hundred additions
    assert torch.allclose(out["cpu"][0], out["cuda"][0], atol=1e-5)
    assert torch.equal(out["cpu"][1], out["cuda"][1]) and out["cpu"][2].tolist() == [20, 20] == out["cuda"][2].tolist()


def test_a_capture_takes_no_pages(monkeypatch):
    import zoo.ops.kvcache as kvcache
    c = PagedKVCache(1, 2, 20, 1, 8, page=4, device="cpu")
    c.reserve(4)
    monkeypatch.setattr(kvcache, "_capturing", lambda t: True)
    c.reserve(4)
    with pytest.raises(RuntimeError, match="before the capture"):
        c.reserve(5)
    assert [len(own) for own in c._pages] == [1, 1]


def test_the_book_on_its_own():
    c = PagedKVCache(1, 2, 20, 1, 8, page=4, device="cpu")
    c.reserve([20, 3])
    assert (c.page_table >= 0).sum(1).tolist() == [5, 1]
    c.release([0])
    assert (c.page_table >= 0).sum(1).tolist() == [0, 1] and len(c._free) == 9
    with pytest.raises(RuntimeError):
        c.reserve(21)
    with pytest.raises(RuntimeError):
        c.replayed(5)


@pytest.mark.gpu
def test_captured_operators_over_long_rows(gpu):
    """Split attention with gathered weights and an eviction that shares out its rows, captured together and replayed
    with other work in between, against eager calls."""
    from test_kvcache import make
    lengths = [18000, 5, 0, 17001]
    q, k, v, table, n = make(4, 2, 4, 64, 128, lengths, torch.bfloat16, "cuda")
    g = torch.Generator("cuda").manual_seed(2)
    scores = torch.rand(k.shape[:3], generator=g, device="cuda")
    positions = torch.randint(0, 18000, k.shape[:3], generator=g, device="cuda", dtype=torch.int32)
    seen = n + 3

    def step(q, k, v, scores, positions):
        o = paged_attention(q, k, v, table, n, scores=scores)
        return o, paged_evict(k, v, scores, positions, table, n, seen, 9000, 500)

    start = [t.clone() for t in (k, v, scores, positions)]
    pools = [t.clone() for t in start]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, *pools)
    torch.cuda.current_stream().wait_stream(side)
    x = q.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, new = step(x, *pools)
    for i in range(5):
        fresh = q * (0.5 + 0.25 * i)
        for a, b in zip(pools, start):
            a.copy_(b)
        x.copy_(fresh)
        graph.replay()
        junk = torch.randn(1024, 1024, device="cuda").sum()
        eager = [t.clone() for t in start]
        want, want_n = step(fresh, *eager)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(new, want_n) and want_n.tolist() == [9000, 5, 0, 9000]
        for a, b in zip(pools, eager):
            assert torch.equal(a.nan_to_num() if a.is_floating_point() else a, b.nan_to_num() if b.is_floating_point() else b)
    assert torch.isfinite(junk)


def test_a_captured_step_sees_the_whole_table(monkeypatch):
    import zoo.ops.kvcache as kvcache
    c = PagedKVCache(1, 2, 40, 1, 8, page=4, device="cpu")
    few = PagedKVCache(1, 2, 40, 1, 8, page=4, pages=3, device="cpu")
    for x in (c, few):
        x.reserve(4)
        assert x._table().shape == (2, 1)
    monkeypatch.setattr(kvcache, "_capturing", lambda t: True)
    assert c._table().shape == (2, 10) and few._table().shape == (2, 3)      # no row can ever have more
    assert c._table().data_ptr() == c.page_table.data_ptr()


@pytest.mark.gpu
def test_captured_step_of_rows_that_come_and_go(gpu):
    """After the capture a row leaves and a prompt longer than any before takes its place, and rows take pages as they
    grow: the replays go on as eager steps do."""
    t = layer("cuda", blocks=2)
    tok, pos = ids(3, 60, "cuda")
    caches = [t.init_cache(3, max_length=70, page=4) for _ in range(2)]
    for c in caches:
        t.prefill([tok[:, :6], pos[:, :6]], c)
    eager, static = caches
    x, p = tok[:, 6].clone(), pos[:, 6].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    spare = t.init_cache(3, max_length=70, page=4)
    with torch.cuda.stream(side):
        t.decode([x, p], spare)
    torch.cuda.current_stream().wait_stream(side)
    static.reserve(1)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = t.decode([x, p], static)
    g.replay()
    assert torch.equal(y, t.decode([x, p], eager))
    at = [7, 7, 7]
    for i in range(30):
        if i == 3:
            for c in caches:
                c.release([1])
                t.prefill([tok[1:2, :31], pos[1:2, :31]], c, rows=[1])
            at[1] = 31
        x.copy_(torch.stack([tok[b, at[b]] for b in range(3)]))
        p.copy_(torch.stack([pos[b, at[b]] for b in range(3)]))
        static.reserve(1)
        g.replay()
        static.replayed(1)
        junk = torch.randn(512, 512, device="cuda") @ torch.randn(512, 512, device="cuda")
        want = t.decode([x, p], eager)
        at = [n + 1 for n in at]
        assert torch.equal(y, want), i
        assert static.lengths.tolist() == eager.lengths.tolist() == at == static._slots
    assert torch.isfinite(junk).all()


def test_the_book_of_replays_counts_the_token_before_its_eviction():
    c = PagedKVCache(1, 1, 20, 1, 8, page=4, budget=4, device="cpu")
    c.reserve(4)
    c._slots = [4]
    with pytest.raises(RuntimeError, match="reserved"):
        c.replayed(1, evicts=True)          # its token had no page
    assert c._slots == [4]
    c.reserve(1)
    c.replayed(1, evicts=True)
    assert c._slots == [4] and len(c._pages[0]) == 2


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("slack", [0, 3, 8])
def test_a_rows_eviction_is_its_own(dev, slack):
    """Rows of unequal length in one cache keep what each keeps alone: a row is cut when it is itself past budget +
    slack."""
    t = layer(dev, blocks=1)
    tok, pos = ids(3, 40, dev)
    first = [6, 11, 2]

    def run(rows):
        c = t.init_cache(len(rows), max_length=40, page=4, budget=8, recent=2, slack=slack)
        n = max(first[b] for b in rows)
        t.prefill([tok[rows, :n], pos[rows, :n]], c, counts=[first[b] for b in rows])
        out = []
        for i in range(14):
            at = [first[b] + i for b in rows]
            y = t.decode([torch.stack([tok[b, a] for b, a in zip(rows, at)]),
                          torch.stack([pos[b, a] for b, a in zip(rows, at)])], c)
            assert c.lengths.tolist() == c._slots and all(n <= 8 + slack for n in c._slots)
            held = []
            for j, n in enumerate(c._slots):
                where = [(int(c.page_table[j, s // 4]), s % 4) for s in range(n)]
                held.append([sorted(int(c.positions[p, h, r]) for p, r in where) for h in range(4)])
            out.append((y, list(c._slots), held))
        return out
    batch = run([0, 1, 2])
    for b in range(3):
        for (y, slots, held), (y1, slots1, held1) in zip(batch, run([b])):
            assert slots[b] == slots1[0] and torch.isfinite(y.float()).all()
            if dev == "cpu":    # products of other batch sizes round otherwise on the GPU, which may turn a close choice
                near(y[b], y1[0], dev)
                assert held[b] == held1[0]


@pytest.mark.parametrize("dev", DEVS)
def test_a_row_that_waits_is_not_cut(dev):
    """A prompt past the budget has gathered no weight before its first step: steps of other rows leave it whole."""
    t = layer(dev, blocks=1)
    tok, pos = ids(3, 40, dev)
    c = t.init_cache(3, max_length=40, page=4, budget=8, recent=2)
    t.prefill([tok[:, :20], pos[:, :20]], c, counts=[20, 8, 3])
    own = list(c._pages[0])
    t.decode([tok[1:, 20], pos[1:, 20]], c, rows=[1, 2])
    assert c._slots == [20, 8, 4] == c.lengths.tolist() and c.seen.tolist() == [20, 9, 4] and c._pages[0] == own
    t.decode([tok[[2, 1], 21], pos[[2, 1], 21]], c, rows=[2, 1])
    assert c._slots == [20, 8, 5] == c.lengths.tolist() and c.seen.tolist() == [20, 10, 5]
    where = [(int(c.page_table[0, s // 4]), s % 4) for s in range(20)]
    assert [int(c.positions[p, 0, r]) for p, r in where] == list(range(20))
    t.decode([tok[:1, 20], pos[:1, 20]], c, rows=[0])
    assert c._slots == [8, 8, 5] == c.lengths.tolist() and len(c._pages[0]) == 3
    used = [p for pages in c._pages for p in pages]
    assert len(used) == len(set(used)) and not set(used) & set(c._free)
    c.evict()
    assert c._slots == [8, 8, 5]


def test_rows_are_counted_from_either_end_and_named_once():
    t = layer("cpu")
    tok, pos = ids(3, 10, "cpu")
    a, b = t.init_cache(3, page=4), t.init_cache(3, page=4)
    for c, rows in ((a, [2, 0]), (b, [-1, 0])):
        t.prefill([tok[:2], pos[:2]], c, rows=rows)
        y = t.decode([tok[:2, 0], pos[:2, 0]], c, rows=rows)
        assert c._slots == [11, 0, 11] == c.lengths.tolist() == c.seen.tolist()
    assert torch.equal(a.page_table, b.page_table) and torch.equal(a.k, b.k) and torch.isfinite(y).all()
    free = list(b._free)
    for call in (lambda: t.decode([tok[:2, 0], pos[:2, 0]], b, rows=[2, -1]),
                 lambda: t.prefill([tok[:2], pos[:2]], b, rows=[1, -2]),
                 lambda: b.reserve(3, [1, -2]), lambda: b.reserve([1, 2], [1]), lambda: b.reserve([1, 1]),
                 lambda: b.reserve([1, -1, 1]), lambda: b.reserve(-1),
                 lambda: b.advance([1, 1], b.lengths), lambda: b.advance(1, b.lengths[:2], [0, 0])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: t.decode([tok[:1, 0], pos[:1, 0]], b, rows=[3]), lambda: b.reserve(1, [-4])):
        with pytest.raises(IndexError):
            call()
    assert b._slots == [11, 0, 11] == b.lengths.tolist() == b.seen.tolist() and b._free == free


def test_a_refused_prompt_takes_no_pages():
    t = layer("cpu")
    tok, pos = ids(2, 10, "cpu")
    both = TransformerLayer.init(vocab=80, seq_len=8, n_block=1, hidden_size=16, n_head=2, bidirectional=True).eval()
    c, d = t.train().init_cache(2, page=4), both.init_cache(2, max_length=12, page=4)
    for run, cache, x in ((t, c, [tok, pos]), (both, d, [tok % 8, pos % 8])):
        free = list(cache._free)
        for call in (lambda: run.prefill(x, cache), lambda: run.decode([x[0][:, 0], x[1][:, 0]], cache)):
            with pytest.raises(RuntimeError):
                call()
        assert cache._free == free and not (cache.page_table >= 0).any()


def test_a_capture_takes_all_rows_one_token_each(monkeypatch):
    """Row numbers and counts come from the host: a captured step cannot take them, and says so before it records."""
    import zoo.ops.kvcache as kvcache
    t = layer("cpu")
    tok, pos = ids(2, 10, "cpu")
    c = t.init_cache(2, max_length=12, page=4)
    c.reserve(2)
    monkeypatch.setattr(kvcache, "_capturing", lambda x: True)
    for call in (lambda: t.decode([tok[:1, 0], pos[:1, 0]], c, rows=[1]), lambda: t.prefill([tok[:, :2], pos[:, :2]], c),
                 lambda: c.evict([0]), lambda: c.advance(1, c.lengths[:1] + 1, [0]), lambda: c.release([0])):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            call()
    assert c._slots == [0, 0] == c.lengths.tolist() and [len(p) for p in c._pages] == [1, 1]
    t.decode([tok[:, 0], pos[:, 0]], c)
    assert c._slots == [1, 1]


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("D,page,budget", [(16, 8, None), (64, 16, None), (128, 64, None), (128, 7, 30), (64, 16, 24)])
def test_attention_over_the_cache_against_64_bits(dev, D, page, budget):
    """A layer's part of the pools as prompts, steps of all and of some rows, and evictions leave it: attention agrees with
    the definition to the tolerance of the operator, and a missing token or even weights would not."""
    from test_kvcache import close, define
    H, layers, rows = 3, 2, [0, 2]
    c = PagedKVCache(layers, 3, 60, H, D, page=page, budget=budget, recent=4 if budget else None, device=dev)
    g = torch.Generator().manual_seed(7)
    kv = torch.randn(layers, 3, 40, 2, H, D, generator=g).to(c.k.dtype).to(dev)
    q = (torch.randn(layers, 3, 40, H, D, generator=g) * 1.5).to(c.k.dtype).to(dev)
    fed = [[], [], []]          # tokens of each row, in order

    def step(take, counts, at=None):
        """Appends tokens take .. to the rows and attends with the last one."""
        every = list(range(3)) if at is None else at
        sub = None if at is None else torch.tensor(at, device=dev)
        c.reserve(counts, at)
        n = torch.tensor(counts, dtype=torch.int32, device=dev)
        for i in range(layers):
            x = kv[i, every, take:take + max(counts)]
            new = c.append(i, x[:, :, 0], x[:, :, 1], counts=n, rows=sub)
            o = c.attend(i, q[i, every, take].contiguous(), new, rows=sub)
            kp, vp, _, _ = c.layer(i)
            table = c.page_table[every]
            ref, mag, _ = define(q[i, every, take], kp, vp, table, new.tolist())
            close(o, ref, mag, D)
            if take and budget is None:
                with pytest.raises(AssertionError):         # as if the newest token were missing
                    r, m, _ = define(q[i, every, take], kp, vp, table, (new - 1).tolist())
                    close(o, r, m, D)
                with pytest.raises(AssertionError):         # as if all weights were equal
                    r, m, _ = define(q[i, every, take] * 0, kp, vp, table, new.tolist())
                    close(o, r, m, D)
                for j, b in enumerate(every):               # what lies in the slots is what was given
                    t = torch.tensor(fed[b] + list(range(take, take + counts[j])), device=dev)
                    where = [(int(table[j, s // page]), s % page) for s in range(len(t))]
                    assert torch.equal(torch.stack([kp[p, :, r] for p, r in where]), kv[i, b, t, 0])
                    assert torch.equal(torch.stack([vp[p, :, r] for p, r in where]), kv[i, b, t, 1])
        c.advance(counts, new, at)
        for j, b in enumerate(every):
            fed[b] += range(take, take + counts[j])

    step(0, [20, 11, 1])
    for take in range(20, 26):
        step(take, [1, 1, 1])
    for take in range(26, 30):
        step(take, [1, 1], rows)
    for take in range(30, 36):
        step(take, [1, 1, 1])
    seen = [len(f) for f in fed]
    assert c.seen.tolist() == seen
    assert c.lengths.tolist() == [min(n, budget or n) for n in seen] == c._slots


def test_a_captured_eviction_sees_the_pages_of_the_steady_state(monkeypatch):
    """A table of all pages would cost a captured eviction what rows of max_length do. Rows past it are cut by replayed()."""
    import zoo.ops.kvcache as kvcache
    widths = []
    real = kvcache.paged_evict
    monkeypatch.setattr(kvcache, "paged_evict", lambda *a, **kw: widths.append(a[4].shape) or real(*a, **kw))
    t = layer("cpu", blocks=1)
    tok, pos = ids(3, 40, "cpu")
    c = t.init_cache(3, max_length=200, page=4, budget=8, recent=2, slack=1)
    t.prefill([tok[:, :20], pos[:, :20]], c, counts=[20, 9, 12])
    c.reserve(1)
    with monkeypatch.context() as m:
        m.setattr(kvcache, "_capturing", lambda x: True)
        t.decode([tok[:, 20], pos[:, 20]], c)
    assert widths == [(3, 3)] and c._slots == [21, 8, 13] == c.lengths.tolist()
    for step in range(2):       # a replay: rows 1 and 2 take a token each, by hand as the graph would do it
        c.reserve(1)
        c.lengths += 1
        c.seen += 1
        with monkeypatch.context() as m:
            m.setattr(kvcache, "_capturing", lambda x: True)
            slots, c._slots = c._slots, [n + 1 for n in c._slots]
            c.evict()
            c._slots = slots
        c.replayed(1, evicts=True)
        assert c._slots == [[8, 9, 8], [9, 8, 9]][step] == c.lengths.tolist()
    assert all(len(own) <= 3 for own in c._pages)


@pytest.mark.gpu
def test_captured_step_with_a_budget_and_rows_that_come_and_go(gpu):
    """Prompts past the budget in rows that were released: the replays and replayed() leave what eager steps leave."""
    t = layer("cuda", blocks=2)
    tok, pos = ids(3, 80, "cuda")
    caches = [t.init_cache(3, max_length=120, page=4, budget=10, recent=3, slack=2) for _ in range(2)]
    for c in caches:
        t.prefill([tok[:, :14], pos[:, :14]], c)
        t.decode([tok[:, 14], pos[:, 14]], c)
        for i in (15, 16):
            t.decode([tok[:, i], pos[:, i]], c)
    eager, static = caches
    assert eager._slots == [12] * 3
    x, p = tok[:, 17].clone(), pos[:, 17].clone()
    static.reserve(1)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = t.decode([x, p], static)
    g.replay()
    assert torch.equal(y, t.decode([x, p], eager))
    at = [18, 18, 18]
    for i in range(30):
        if i in (3, 20):
            b = 1 if i == 3 else 2
            for c in caches:
                c.release([b])
                t.prefill([tok[b:b + 1, :41 + i], pos[b:b + 1, :41 + i]], c, rows=[b])
            at[b] = 41 + i
        x.copy_(torch.stack([tok[b, at[b]] for b in range(3)]))
        p.copy_(torch.stack([pos[b, at[b]] for b in range(3)]))
        static.reserve(1)
        g.replay()
        static.replayed(1, evicts=True)
        want = t.decode([x, p], eager)
        at = [n + 1 for n in at]
        assert torch.equal(y, want), i
        assert static.lengths.tolist() == eager.lengths.tolist() == eager._slots == static._slots
        assert static.seen.tolist() == eager.seen.tolist() == at
        assert [len(own) for own in static._pages] == [len(own) for own in eager._pages]
    for b in range(3):
        for s in range(eager._slots[b]):
            e, f = int(eager.page_table[b, s // 4]), int(static.page_table[b, s // 4])
            assert torch.equal(eager.positions[e, :, s % 4], static.positions[f, :, s % 4])
            assert torch.equal(eager.k[e, :, s % 4], static.k[f, :, s % 4])
