"""The paged key/value cache (zoo.ops.kvcache, csrc/kernels/kvcache.hip) against its definition in 64 bits,
written slot by slot here.

Tolerances. The attention output is rounded once to the cache's type: half a step, eps / 2 of the value. Before
that everything is float32: the products q.k over D dims and the sums over n slots. With logits |s| <= 20, a
logit is off by at most 20 (D + 3) 2^-24 in the worst order of summation, about sqrt(D) of these in practice; a
weight by twice that relative; the weights' two-part 16-bit split by 2^-16 (bfloat16) or 2^-21 (float16). So an
output is off by at most eps / 2 |o| + (twice the split + 2^-24 * 40 * (D + 3)) * sum_j w_j |v_j|; gathered weights by
2^-24 * 40 * (D + 3) times the weight plus half a step of the score.
"""
import math

import pytest
import torch

from zoo.ops import paged_append, paged_attention, paged_evict

GPU = pytest.mark.gpu
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


def make(B, H, G, D, page, lengths, dtype, dev, seed=0, order="phsd", spare=3, width=None, junk=float("nan")):
    """A cache whose sequences own scattered pages; rows nobody uses hold `junk`."""
    g = torch.Generator().manual_seed(seed)
    own = [-(-n // page) for n in lengths]
    width = max([1] + own) if width is None else width
    P = sum(own) + spare
    ids = torch.randperm(P, generator=g)
    table = torch.full((B, width), -7, dtype=torch.int32)
    k, v = (torch.full((P, H, page, D), junk) for _ in range(2))
    at = 0
    for b, n in enumerate(lengths):
        for i in range(own[b]):
            p = int(ids[at])
            at += 1
            table[b, i] = p
            rows = min(page, n - i * page)
            k[p, :, :rows] = torch.randn(H, rows, D, generator=g)
            v[p, :, :rows] = torch.randn(H, rows, D, generator=g)
    q = torch.randn(B, H * G, D, generator=g) * 1.5

    def lay(t):
        t = t.to(dtype)
        if order == "pshd":      # [pages, page, heads, dim] in memory
            t = t.transpose(1, 2).contiguous().transpose(1, 2)
        return t.to(dev) if order == "phsd" else _keep(t, dev)

    def _keep(t, dev):
        if dev == "cpu":
            return t
        return t.transpose(1, 2).to(dev).transpose(1, 2)
    return q.to(dtype).to(dev), lay(k), lay(v), table.to(dev), torch.tensor(lengths, dtype=torch.int32, device=dev)


def define(q, k, v, table, lengths, scale=None):
    """o, sum_j w_j |v_j| and the weights [B][H, n], in float64 on the CPU."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    B, Hq, D = q.shape
    H, page = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(D) if scale is None else scale
    o, mag, ws = torch.zeros(B, Hq, D).double(), torch.zeros(B, Hq, D).double(), []
    for b in range(B):
        n = int(lengths[b])
        slots = [(int(table[b, s // page]), s % page) for s in range(n)]
        w_b = torch.zeros(H, n).double()
        for h in range(H if n else 0):
            kk = torch.stack([k[p, h, r] for p, r in slots])
            vv = torch.stack([v[p, h, r] for p, r in slots])
            for g in range(Hq // H):
                i = h * (Hq // H) + g
                w = torch.softmax(kk @ q[b, i] * scale, 0)
                o[b, i] = w @ vv
                mag[b, i] = w @ vv.abs()
                w_b[h] += w
        ws.append(w_b)
    return o, mag, ws


def close(o, ref, mag, D):
    eps = torch.finfo(o.dtype).eps
    split = {BF: 2.0 ** -15, HF: 2.0 ** -20, FL: 0.0}[o.dtype]
    tol = eps / 2 * ref.abs() + (split + 2.0 ** -24 * 40 * (D + 3)) * mag + 1e-30
    if o.dtype == HF:
        tol = tol + 2.0 ** -25      # half a step of its subnormal numbers
    err = (o.double().cpu() - ref).abs()
    assert torch.isfinite(o.float()).all()
    assert (err <= tol).all(), (err / tol).max().item()


CASES = [
    # H, G, D, page, dtype, order, lengths
    (1, 1, 64, 16, BF, "phsd", [1]),
    (12, 1, 64, 16, BF, "phsd", [77]),
    (3, 1, 64, 64, BF, "pshd", [0, 1, 63, 64, 65, 200]),
    (2, 4, 128, 16, BF, "phsd", [513, 0, 31, 32, 33, 129, 1]),
    (2, 4, 128, 16, HF, "pshd", [513, 0, 31, 32, 33, 129, 1]),
    (2, 8, 128, 64, FL, "phsd", [300, 17, 0, 16]),
    (1, 16, 256, 32, BF, "phsd", [700, 5]),
    (2, 3, 256, 32, FL, "phsd", [130, 5, 16]),
    (1, 24, 64, 48, HF, "phsd", [900, 20]),          # two blocks of query heads
    (2, 71, 64, 16, BF, "phsd", [100, 300]),         # five of them
    (1, 2, 16, 24, BF, "phsd", [500, 3]),
    (2, 17, 128, 64, BF, "phsd", [700, 1, 0]),
    (1, 32, 256, 16, HF, "phsd", [600, 33]),
    (1, 40, 200, 16, FL, "phsd", [300, 15]),
    (1, 33, 96, 32, BF, "pshd", [1200, 64]),
    (1, 32, 72, 11, FL, "phsd", [900, 12]),
    (1, 256, 64, 16, BF, "phsd", [2100, 40]),
    (2, 24, 24, 16, HF, "phsd", [2600, 40, 700]),
    (2, 1, 40, 7, BF, "phsd", [400, 0, 6, 7, 8]),    # no multiple of 16 in sight
    (2, 5, 80, 1, HF, "phsd", [270, 4]),
    (3, 2, 96, 100, FL, "pshd", [410, 99, 100, 101]),
    (2, 2, 200, 33, BF, "phsd", [290, 64]),
    (1, 1, 8, 5, FL, "phsd", [37]),
    (1, 4, 128, 128, BF, "phsd", [5000]),            # split over many workgroups
    (2, 2, 128, 20, HF, "phsd", [3000, 1, 0, 0, 40]),
]


def _check_attention(dev, H, G, D, page, dtype, order, lengths, weights):
    q, k, v, table, n = make(len(lengths), H, G, D, page, lengths, dtype, dev, order=order)
    ref, mag, ws = define(q, k, v, table, lengths)
    if not weights:
        close(paged_attention(q, k, v, table, n), ref, mag, D)
        return
    start = torch.rand(k.shape[:3]).to(dev)
    out = torch.full_like(start, -3.0)
    close(paged_attention(q, k, v, table, n, scores=start, scores_out=out), ref, mag, D)
    want = torch.full(k.shape[:3], -3.0).double()     # slots behind the last keep what they held
    tol = torch.zeros(k.shape[:3]).double()
    for b, m in enumerate(lengths):
        for s in range(m):
            at = (int(table[b, s // page]), slice(None), s % page)
            want[at] = start[at].double().cpu() + ws[b][:, s]
            tol[at] = 2.0 ** -24 * 40 * (D + 3) * ws[b][:, s] + 2.0 ** -24 * want[at]
    assert ((out.double().cpu() - want).abs() <= tol + 1e-30).all()
    # in place: the same sums
    paged_attention(q, k, v, table, n, scores=start)
    used = want != -3.0
    assert torch.equal(start.cpu()[used], out.cpu()[used])


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("H,G,D,page,dtype,order,lengths", CASES[:16])
def test_attention_cpu(H, G, D, page, dtype, order, lengths, weights):
    _check_attention("cpu", H, G, D, page, dtype, order, lengths, weights)


@GPU
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("H,G,D,page,dtype,order,lengths", CASES)
def test_attention_gpu(gpu, H, G, D, page, dtype, order, lengths, weights):
    _check_attention("cuda", H, G, D, page, dtype, order, lengths, weights)


# ---------------------------------------------------------------------------- values that arithmetic must not touch
def _check_odd_values(dev, dtype=BF):
    q, k, v, table, n = make(3, 2, 2, 64, 16, [40, 33, 20], dtype, dev)
    # a key that makes one logit -inf: weight 0, and the others as if it were not there
    p, r = int(table[0, 1]), 3
    k[p, 0, r] = 0
    k[p, 0, r, 5] = -math.inf
    q[0, :2, 5] = 1.0
    ref, mag, _ = define(q, k, v, table, [40, 33, 20])
    assert torch.isfinite(ref[0, :2]).all()
    o = paged_attention(q, k, v, table, n)
    close(o, ref, mag, 64)
    # an infinite value with weight comes through, a NaN key makes its heads NaN and no other
    v[int(table[1, 0]), 1, 2, 7] = math.inf
    k[int(table[2, 0]), 1, 4, 9] = math.nan
    o = paged_attention(q, k, v, table, n).float().cpu()
    assert o[1, 2, 7] == math.inf and o[1, 3, 7] == math.inf and torch.isfinite(o[1, :2]).all()
    assert torch.isnan(o[2, 2:]).all() and torch.isfinite(o[2, :2]).all()
    # huge logits: all weight on one slot
    q2 = q * (1e4 if dtype != HF else 1e3)
    ref, mag, _ = define(q2[:1, :2], k[:, :1], v[:, :1], table[:1], [40])
    o = paged_attention(q2, k, v, table, n)
    assert (o[0, :2].double().cpu() - ref[0]).abs().max() <= 2.0 ** -7 * ref.abs().max()


def test_odd_values_cpu():
    _check_odd_values("cpu")


@GPU
@pytest.mark.parametrize("dtype", [BF, HF, FL])
def test_odd_values_gpu(gpu, dtype):
    _check_odd_values("cuda", dtype)


def _check_bad(dev):
    """Lengths and pages that point nowhere: NaN for that sequence, nothing written, the others unharmed."""
    lengths = [40, 33, 20, 70]
    q, k, v, table, n = make(4, 2, 2, 64, 16, lengths, BF, dev)
    good = paged_attention(q, k, v, table, n)
    for what in ("page", "negative page", "long", "negative"):
        t2, n2 = table.clone(), n.clone()
        if what == "page":
            t2[1, 2] = k.shape[0]
        elif what == "negative page":
            t2[1, 0] = -1
        else:
            n2[1] = 16 * table.shape[1] + 1 if what == "long" else -1
        o = paged_attention(q, k, v, t2, n2)
        assert torch.isnan(o[1]).all(), what
        assert torch.equal(o[[0, 2, 3]], good[[0, 2, 3]]), what
        pools = [k.clone(), v.clone(), torch.rand(k.shape[:3]).to(dev), torch.randint(0, 70, k.shape[:3]).int().to(dev)]
        before = [x.clone() for x in pools]
        kk = torch.randn(4, 1, 2, 64).to(BF).to(dev)
        if what in ("long", "negative"):
            new = paged_append(kk[1:2], kk[1:2], pools[0], pools[1], t2[1:2], n2[1:2], scores=pools[2], positions=pools[3])
            assert torch.equal(new, n2[1:2])
        else:
            n3 = torch.tensor([32 if what == "page" else 0], dtype=torch.int32, device=dev)
            new = paged_append(kk[1:2], kk[1:2], pools[0], pools[1], t2[1:2], n3, scores=pools[2], positions=pools[3])
            assert torch.equal(new, n3 + 1)
        new = paged_evict(*pools, t2[1:2], n2[1:2], n2[1:2].clone(), 10, 2)
        assert torch.equal(new, n2[1:2])
        for x, y in zip(pools, before):
            assert torch.equal(x.nan_to_num(), y.nan_to_num()), what
    # longer than the bound that the caller gave
    o = paged_attention(q, k, v, table, n, max_length=40)
    assert torch.isnan(o[3]).all() and torch.equal(o[:3], good[:3])


def test_bad_lengths_and_pages_cpu():
    _check_bad("cpu")


@GPU
def test_bad_lengths_and_pages_gpu(gpu):
    _check_bad("cuda")


@GPU
def test_append_past_the_table_gpu(gpu):
    _past_the_table("cuda")


def test_append_past_the_table_cpu():
    _past_the_table("cpu")


def _past_the_table(dev):
    q, k, v, table, n = make(2, 1, 1, 8, 4, [6, 3], FL, dev, width=2)
    table[1, 1] = int(k.shape[0]) - 1 if int(k.shape[0]) - 1 not in table.tolist()[0] + table.tolist()[1] else _free(table, k)
    new_k, new_v = torch.randn(2, 1, 2, 5, 1, 8).to(dev)[:, 0]
    k0 = k.clone()
    new = paged_append(new_k, new_v, k, v, table, n)
    assert new.tolist() == [11, 8]
    written = {(int(table[0, 1]), 2): (0, 0), (int(table[0, 1]), 3): (0, 1)}
    for t in range(5):
        written[(int(table[1, (3 + t) // 4]), (3 + t) % 4)] = (1, t)
    for p in range(k.shape[0]):
        for r in range(4):
            src = written.get((p, r))
            want = k0[p, :, r] if src is None else new_k[src[0], src[1]]
            assert torch.equal(k[p, :, r].nan_to_num(), want.nan_to_num())
    assert torch.isnan(paged_attention(q, k, v, table, new)[0]).all()


def _free(table, k):
    return next(p for p in range(k.shape[0]) if p not in set(table.flatten().tolist()))


# ---------------------------------------------------------------------------- append
@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=GPU)])
@pytest.mark.parametrize("H,D,page,T,dtype,order,counted", [
    (12, 64, 16, 1, BF, "phsd", False), (2, 128, 64, 33, HF, "pshd", True), (3, 8, 7, 20, FL, "phsd", True),
    (1, 256, 1, 5, FL, "pshd", True), (5, 40, 24, 100, BF, "phsd", True), (2, 16, 16, 0, BF, "phsd", False)])
def test_append(dev, H, D, page, T, dtype, order, counted):
    lengths = [0, 5, page, 2 * page - 1, 31]
    counts = [T, 0, max(T - 1, 0), min(1, T), T + 9] if counted else [T] * 5       # more than there are: all of them
    real = [max(0, min(T, c)) for c in counts]
    q, k, v, table, _ = make(5, H, 1, D, page, [a + b for a, b in zip(lengths, real)], dtype, dev, order=order, junk=2.0)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    seen = n + 100
    qkv = torch.randn(5, T, 3, H, D).to(dtype).to(dev)
    new_k, new_v = qkv[:, :, 1], qkv[:, :, 2]
    scores, positions = torch.rand(k.shape[:3]).to(dev), torch.zeros(k.shape[:3]).int().to(dev)
    want = [t.clone() for t in (k, v, scores, positions)]
    for b in range(5):
        for t in range(real[b]):
            s = lengths[b] + t
            at = (int(table[b, s // page]), slice(None), s % page)
            want[0][at], want[1][at], want[2][at], want[3][at] = new_k[b, t], new_v[b, t], 0.0, lengths[b] + 100 + t
    c = torch.tensor(counts, dtype=torch.int32, device=dev) if counted else None
    got = paged_append(new_k, new_v, k, v, table, n, counts=c, seen=seen, scores=scores, positions=positions)
    assert got.tolist() == [a + b for a, b in zip(lengths, real)]
    assert n.tolist() == lengths
    for x, y in zip((k, v, scores, positions), want):
        assert torch.equal(x, y)
    positions.zero_()
    paged_append(new_k, new_v, k, v, table, n, counts=c, positions=positions)       # by default the slot is the position
    for b in range(5):
        for t in range(real[b]):
            s = lengths[b] + t
            assert (positions[int(table[b, s // page]), :, s % page] == s).all()


# ---------------------------------------------------------------------------- evict
def evict_by_definition(pools, table, lengths, seen, budget, recent):
    k, v, scores, positions = (t.clone() for t in pools)
    H, page = k.shape[1], k.shape[2]
    sc, po = scores.cpu(), positions.cpu()
    for b, n in enumerate(lengths):
        at = [(int(table[b, s // page]), s % page) for s in range(n)]
        for h in range(H if n > budget else 0):
            rank = []
            for s, (p, r) in enumerate(at):
                x = float(sc[p, h, r])
                late = int(po[p, h, r]) >= seen[b] - recent
                rank.append((0 if late else 2 if math.isnan(x) else 1, 0.0 if late or math.isnan(x) else -x, s))
            kept = {s for _, _, s in sorted(rank)[:budget]}
            holes = [s for s in range(budget) if s not in kept]
            behind = [s for s in sorted(kept) if s >= budget]
            for d, s in zip(holes, behind):
                for t in (k, v, scores, positions):
                    t[at[d][0], h, at[d][1]] = t[at[s][0], h, at[s][1]]
    return k, v, scores, positions


EVICT_LONG = [      # rows shared out over workgroups
    (1, 8, 64, FL, "phsd", [40000, 17, 9000], 6000, 100, "ties"),
    (2, 8, 100, BF, "pshd", [20000, 8193, 4096, 0], 4096, 0, "plain"),
    (1, 16, 128, BF, "phsd", [17000], 16999, 16999, "odd"),
    (1, 8, 7, FL, "phsd", [30000, 12345], 12345, 77, "zeros"),
]


@GPU
@pytest.mark.parametrize("H,D,page,dtype,order,lengths,budget,recent,kind", EVICT_LONG)
def test_evict_long(gpu, H, D, page, dtype, order, lengths, budget, recent, kind):
    test_evict("cuda", H, D, page, dtype, order, lengths, budget, recent, kind)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=GPU)])
@pytest.mark.parametrize("H,D,page,dtype,order,lengths,budget,recent,kind", [
    (2, 64, 16, BF, "phsd", [100, 0, 50, 51, 1], 50, 10, "plain"),
    (1, 8, 7, FL, "pshd", [60, 20, 13], 1, 0, "plain"),
    (3, 40, 24, HF, "phsd", [400, 399, 25], 24, 24, "ties"),
    (2, 64, 1, BF, "phsd", [70, 64], 63, 1, "odd"),
    (2, 128, 64, BF, "pshd", [513, 514, 512], 512, 128, "plain"),
    (2, 16, 33, FL, "phsd", [1500, 1100, 1025], 700, 5, "ties"),
    (1, 8, 128, BF, "phsd", [2500], 2048, 0, "zeros"),
    (2, 8, 16, FL, "phsd", [300], 100, 50, "twice"),
    (1, 8, 16, FL, "phsd", [30], 1000, 3, "plain"),
    (2, 8, 16, FL, "phsd", [24, 23, 22, 21, 25], 20, 0, "ties"),      # a few over the budget
    (2, 8, 16, FL, "phsd", [104, 103, 102, 101, 105], 100, 9, "zeros"),
    (3, 8, 5, FL, "pshd", [3, 4, 5, 2], 1, 0, "odd"),
    (1, 8, 64, BF, "phsd", [3003, 3001], 3000, 3000, "odd"),
])
def test_evict(dev, H, D, page, dtype, order, lengths, budget, recent, kind):
    B = len(lengths)
    _, k, v, table, n = make(B, H, 1, D, page, lengths, dtype, dev, order=order, junk=2.0)
    g = torch.Generator().manual_seed(5)
    shape = k.shape[:3]
    scores = torch.rand(shape, generator=g)
    if kind == "ties":
        scores = (scores * 4).floor() / 4
    elif kind == "zeros":
        scores.zero_()
    elif kind == "odd":
        special = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-42, -1e-42, -3.0])
        scores = special[torch.randint(0, 8, shape, generator=g)]
    positions = torch.zeros(shape, dtype=torch.int32)
    for b, m in enumerate(lengths):
        for h in range(H):
            order_ = torch.randperm(m, generator=g) if kind != "twice" else torch.randint(0, m, (m,), generator=g)
            for s in range(m):
                positions[int(table[b, s // page]), h, s % page] = int(order_[s])
    scores, positions = scores.to(dev), positions.to(dev)
    seen = torch.tensor(lengths, dtype=torch.int32, device=dev)
    want = evict_by_definition((k, v, scores, positions), table, lengths, lengths, budget, recent)
    # out of place: scores and positions of the kept slots in new pools, nothing else there
    k2, v2 = k.clone(), v.clone()
    so, po = torch.full_like(scores, -5.0), torch.full_like(positions, -5)
    got = paged_evict(k2, v2, scores, positions, table, n, seen, budget, recent, scores_out=so, positions_out=po)
    assert got.tolist() == [min(m, budget) for m in lengths] and n.tolist() == lengths
    assert torch.equal(k2, want[0]) and torch.equal(v2, want[1])
    used = torch.zeros(shape, dtype=torch.bool)
    for b, m in enumerate(lengths):
        for s in range(min(m, budget)):
            used[int(table[b, s // page]), :, s % page] = True
    used = used.to(dev)
    assert torch.equal(so[used].view(torch.int32), want[2][used].view(torch.int32)) and torch.equal(po[used], want[3][used])
    assert (so[~used] == -5.0).all() and (po[~used] == -5).all()
    # in place
    got = paged_evict(k, v, scores, positions, table, n, seen, budget, recent)
    assert got.tolist() == [min(m, budget) for m in lengths]
    for x, y in zip((k, v, scores, positions), want):
        assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))


# ---------------------------------------------------------------------------- refusals
@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=GPU)])
def test_refusals(dev):
    q, k, v, table, n = make(2, 2, 2, 16, 8, [9, 5], BF, dev)
    s, p = torch.zeros(k.shape[:3]).to(dev), torch.zeros(k.shape[:3]).int().to(dev)
    x = torch.zeros(2, 1, 2, 16).to(BF).to(dev)

    def no(f, *a, **kw):
        with pytest.raises((RuntimeError, TypeError)):
            f(*a, **kw)
    no(paged_attention, q[:, :3], k, v, table, n)
    no(paged_attention, q[:1], k, v, table, n)
    no(paged_attention, q[:, :, :8], k, v, table, n)
    no(paged_attention, q, k, v[:, :1], table, n)
    no(paged_attention, q, k, v, table.long(), n)
    no(paged_attention, q, k, v, table, n.long())
    no(paged_attention, q, k, v, table, n[:1])
    no(paged_attention, q, k, v, table, n, scale=math.inf)
    no(paged_attention, q, k, v, table, n, scores_out=s)
    no(paged_attention, q, k, v, table, n, max_length=-1)
    no(paged_attention, q.float().requires_grad_(), k.float(), v.float(), table, n)
    no(paged_attention, q, k, v, table, n, scores=s.clone().requires_grad_())
    no(paged_append, x.clone().requires_grad_(), x, k, v, table, n)
    no(paged_evict, k, v, s.clone().requires_grad_(), p, table, n, n, 4)
    no(paged_append, x[:1], x[:1], k, v, table, n)
    no(paged_append, x[..., :8], x[..., :8], k, v, table, n)
    no(paged_append, x.float(), x.float(), k, v, table, n)
    no(paged_evict, k, v, s, p, table, n, n, 0)
    no(paged_evict, k, v, s, p, table, n, n, 4, 5)
    no(paged_evict, k, v, s, p, table, n, n, 4, -1)
    if dev == "cuda":
        no(paged_attention, q.half(), k, v, table, n)
        no(paged_attention, q, k, v, table.cpu(), n)
        no(paged_attention, q, k, v, table, n, scores=s[:1])
        no(paged_attention, q, k, v, table, n, scores=s.double())
        no(paged_attention, q, k, v, table, n, scores=s, scores_out=s.expand(4, *s.shape)[0, :1])
        no(paged_attention, q, k.transpose(2, 3).contiguous().transpose(2, 3), v, table, n)
        no(paged_attention, q[..., :12].contiguous(), k[..., :12].contiguous(), v[..., :12].contiguous(), table, n)
        big = torch.zeros(3, 1, 8, 264, dtype=BF, device=dev)
        no(paged_attention, big[:2, 0, :1], big, big, table, n)
        wide = torch.zeros(2, 514, 16, dtype=BF, device=dev)
        no(paged_attention, wide, k, v, table, n)                       # 257 heads to a kv head
        no(paged_append, x, x, k, k, table, n)                          # keys and values in one place
        no(paged_append, x, x, k[:1].expand(k.shape), v, table, n)
        one = table[:1].expand(2, -1)                                   # both rows the same pages
        assert torch.equal(paged_attention(q, k, v, one, n)[0], paged_attention(q, k, v, table, n)[0])
        no(paged_attention, q, k, v, one, n, scores=s)
        no(paged_append, x, x, k, v, one, n)
        no(paged_evict, k, v, s, p, one, n, n, 4)
        no(paged_evict, k, v, s.half(), p, table, n, n, 4)
        no(paged_evict, k, v, s, p.long(), table, n, n, 4)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=GPU)])
@pytest.mark.parametrize("pages,batch,width", [(0, 2, 3), (4, 2, 0), (4, 0, 3), (0, 0, 0)])
def test_nothing_there(dev, pages, batch, width):
    """No pages, no sequences, no room in the table: empty sequences are zeros, and there are no others."""
    k, v = (torch.zeros(pages, 2, 8, 16).to(dev) for _ in range(2))
    s, p = torch.zeros(pages, 2, 8).to(dev), torch.zeros(pages, 2, 8, dtype=torch.int32).to(dev)
    table = torch.zeros(batch, width, dtype=torch.int32).to(dev)
    n = torch.zeros(batch, dtype=torch.int32).to(dev)
    q, new = torch.ones(batch, 4, 16).to(dev), torch.ones(batch, 1, 2, 16).to(dev)
    o = paged_attention(q, k, v, table, n)
    assert tuple(o.shape) == (batch, 4, 16) and not o.any()
    assert not paged_attention(q, k, v, table, n, scores=s).any()
    assert paged_evict(k, v, s, p, table, n, n.clone(), 3, 1).tolist() == [0] * batch
    after = paged_append(new, new, k, v, table, n, scores=s, positions=p)
    assert after.tolist() == [1] * batch
    if batch and (width == 0 or pages == 0):
        assert torch.isnan(paged_attention(q, k, v, table, after)).all()
        assert paged_evict(k, v, s, p, table, after, after.clone(), 3, 1).tolist() == [1] * batch


@GPU
def test_far_pages(gpu):
    """Offsets past 2^31 elements and 2^32 bytes: the last pages of a pool of 5 GiB."""
    P = 5 * 2 ** 30 // (2 * 128 * 128 * 2)
    k = torch.zeros(P, 2, 128, 128, dtype=BF, device="cuda")
    assert k.numel() > 2 ** 31
    near = make(2, 2, 2, 128, 128, [300, 129], BF, "cuda")
    q, kn, vn, table, n = near
    v = torch.zeros_like(k)
    far = torch.where(table >= 0, table + (P - kn.shape[0]), table)
    k[P - kn.shape[0]:], v[P - kn.shape[0]:] = kn, vn
    assert torch.equal(paged_attention(q, k, v, far, n), paged_attention(q, kn, vn, table, n))
    new = torch.randn(2, 3, 2, 128).to(BF).cuda()
    for kk, vv, t in ((k, v, far), (kn, vn, table)):
        s = torch.arange(128, device="cuda").expand(kk.shape[:3]).remainder(37).float().contiguous()
        p = torch.zeros(kk.shape[:3], dtype=torch.int32, device="cuda")
        m = paged_append(new, new, kk, vv, t, n, scores=s, positions=p)
        paged_evict(kk, vv, s, p, t, m, m + 1000, 100, 0)
    a, b = k[P - kn.shape[0]:], v[P - kn.shape[0]:]
    assert torch.equal(a.nan_to_num(), kn.nan_to_num()) and torch.equal(b.nan_to_num(), vn.nan_to_num())
    assert not k[:P - kn.shape[0]].any()


@GPU
def test_many_short_sequences(gpu):
    """More sequences than a wave has lanes, split and unsplit, with bad ones among them."""
    g = torch.Generator().manual_seed(4)
    lengths = torch.randint(0, 900, (300,), generator=g).tolist()
    q, k, v, table, n = make(300, 1, 2, 64, 32, lengths, BF, "cuda")
    o = paged_attention(q, k, v, table, n)
    wide = torch.nn.functional.pad(table, (0, 400), value=-1).contiguous()       # capacity past the unsplit form
    n[7], n[200] = -5, 10 ** 6
    o2 = paged_attention(q, k, v, wide, n)
    assert torch.isnan(o2[[7, 200]]).all()
    fine = [i for i in range(300) if i not in (7, 200)]
    for b in (0, 63, 64, 128, 255, 299):
        ref, mag, _ = define(q[b:b + 1], k, v, table[b:b + 1], lengths[b:b + 1])
        close(o[b:b + 1], ref, mag, 64)
        close(o2[b:b + 1], ref, mag, 64)
    assert torch.isfinite(o2[fine]).all()


@GPU
@pytest.mark.parametrize("longest,rows", [(40, 900), (1000, 45)])
def test_streamed_past_the_caches(gpu, longest, rows):
    """Batches too large for the caches take their keys and values past them, sequences that are one work item each and
    split ones: the same results as row by row."""
    H, D, page = 16, 128, 16
    lengths = [longest - i % 7 for i in range(rows)]
    assert 2 * H * D * 4 * sum(lengths) > 4e8
    width = -(-longest // page)
    g = torch.Generator("cuda").manual_seed(3)
    k, v = (torch.randn(rows * width, H, page, D, generator=g, device="cuda") for _ in range(2))
    table = torch.arange(rows * width, dtype=torch.int32, device="cuda").view(width, rows).t().contiguous()
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = torch.randn(rows, H, D, generator=g, device="cuda")
    o = paged_attention(q, k, v, table, n)
    for b in range(0, rows, rows // 5):
        ref, mag, _ = define(q[b:b + 1], k, v, table[b:b + 1], lengths[b:b + 1])
        close(o[b:b + 1], ref, mag, D)
        close(paged_attention(q[b:b + 1], k, v, table[b:b + 1], n[b:b + 1]), ref, mag, D)


# ---------------------------------------------------------------------------- weights in full
def _cancelling(dev, dtype, lengths_of_two=64, D=64):
    """Two slots whose weighted values cancel but for the rounding of the second value, so that an output is small against
    what it is summed from and shows how exactly the weights were kept. One product makes a logit: it is exact."""
    g = torch.Generator().manual_seed(11)
    B, H = lengths_of_two, 4
    q, k, v, table, n = make(B, H, 1, D, 16, [2] * B, FL, "cpu", seed=1)
    q.zero_()
    q[:, :, 0] = 1.0
    a = (torch.rand(B, H, 2, generator=g) * 2 - 1).to(dtype).float()
    v0 = (torch.randn(B, H, D, generator=g)).to(dtype).float()
    w = torch.softmax(a.double(), -1)
    v1 = (-v0.double() * w[..., :1] / w[..., 1:]).to(dtype).float()
    for b in range(B):
        p = int(table[b, 0])
        k[p, :, :2] = 0.0
        k[p, :, :2, 0] = a[b]
        v[p, :, 0], v[p, :, 1] = v0[b], v1[b]
    return [t.to(dtype).to(dev) for t in (q, k, v)] + [table.to(dev), n.to(dev)]


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=GPU)])
@pytest.mark.parametrize("dtype", [BF, HF, FL])
def test_weights_are_kept_to_float32(dev, dtype):
    """A logit of at most 1 is multiplied by log2(e) and taken off the maximum, 2^-24 relative each, which moves a weight
    by at most 2^-22; its exponential and its place in the sums add 2^-23 each, a split into 16-bit parts at most 2^-22. So
    an output is off by half a step and at most 2^-20 of what it is summed from. (Weights of 16 bits are off by up to
    2^-16, and the values' own rounding leaves outputs of 2^-9 of their parts in bfloat16, whose half step is
    2^-17.)"""
    args = _cancelling(dev, dtype)
    ref, mag, _ = define(*[t.cpu() for t in args[:4]], [2] * 64, scale=1.0)
    o = paged_attention(*args, scale=1.0).double().cpu()
    tol = torch.finfo(dtype).eps / 2 * ref.abs() + 2.0 ** -20 * mag + (2.0 ** -25 if dtype == HF else 0.0)
    assert ((o - ref).abs() <= tol).all(), ((o - ref).abs() / tol).max().item()


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=GPU)])
@pytest.mark.parametrize("dtype,logit", [(BF, -500.0), (HF, -500.0), (FL, -500.0), (BF, -100.0), (HF, -60.0)])
def test_slots_without_weight_add_nothing(dev, dtype, logit):
    """One slot has all the weight and a small value, a thousand others hold the type's largest values and a weight that is 0
    in float32 (exp -500), or too small to count: 1000 e^-100 3e38 is below 1e-2 of 2^-4's half step in
    bfloat16, 1000 e^-60 65504 below 1e-14 of it in float16."""
    n = 1001
    q, k, v, table, lens = make(1, 2, 3, 64, 16, [n], FL, "cpu", seed=2)
    big = torch.finfo(dtype).max if dtype != BF or logit == -500.0 else 2.0 ** 100
    q.zero_()
    q[:, :, 0] = 1.0
    k.zero_()
    k[..., 0] = logit
    v.fill_(big)
    k[int(table[0, 0]), :, 0, 0] = 0.0
    v[int(table[0, 0]), :, 0] = 2.0 ** -4
    q, k, v = (t.to(dtype).to(dev) for t in (q, k, v))
    o = paged_attention(q, k, v, table.to(dev), lens.to(dev), scale=1.0).double().cpu()
    assert ((o - 2.0 ** -4).abs() <= torch.finfo(dtype).eps / 2 * 2.0 ** -4).all(), (o - 2.0 ** -4).abs().max().item()


# ---------------------------------------------------------------------------- weights of a sequence with a bad page
@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=GPU)])
@pytest.mark.parametrize("H,G,D,page,dtype,lengths,width", [
    (2, 2, 64, 16, BF, [40, 33, 20, 70], None),          # one work item each, products in LDS
    (1, 16, 64, 16, BF, [300, 290, 20, 310], None),      # products in memory
    (2, 2, 128, 16, HF, [900, 830, 20, 1200], 400),      # split
    (1, 40, 64, 16, BF, [40, 33, 20, 70], None),         # several blocks of query heads
    (1, 70, 128, 16, BF, [900, 830, 0, 1200], 300),      # ... and split
    (3, 1, 80, 7, FL, [700, 650, 9, 800], 500),
])
def test_bad_pages_leave_the_gathered_weights(dev, H, G, D, page, dtype, lengths, width):
    """A sequence that names a bad page gathers nothing, on its good pages neither; the others do as ever. NaN that the
    data holds comes through."""
    q, k, v, table, n = make(4, H, G, D, page, lengths, dtype, dev, width=width)
    start = torch.rand(k.shape[:3]).to(dev)
    good = torch.full_like(start, -3.0)
    o = paged_attention(q, k, v, table, n, scores=start, scores_out=good)
    rows = [[(int(table[b, s // page]), s % page) for s in range(m)] for b, m in enumerate(lengths)]
    for at, bad in ((0, -1), (1, k.shape[0]), (lengths[1] // page, -5)):
        t2 = table.clone()
        t2[1, at] = bad
        want, kept = good.clone(), start.clone()
        for p, r in rows[1]:
            want[p, :, r] = -3.0
        for b in (0, 2, 3):
            for p, r in rows[b]:
                kept[p, :, r] = good[p, :, r]
        out = torch.full_like(start, -3.0)
        o2 = paged_attention(q, k, v, t2, n, scores=start, scores_out=out)
        assert torch.isnan(o2[1]).all() and torch.equal(o2[[0, 2, 3]], o[[0, 2, 3]])
        assert torch.equal(out, want), at
        here = start.clone()
        paged_attention(q, k, v, t2, n, scores=here)
        assert torch.equal(here, kept), at
    p, r = rows[3][5]
    k[p, 0, r, 3] = float("nan")
    out = torch.full_like(start, -3.0)
    o2 = paged_attention(q, k, v, table, n, scores=start, scores_out=out)
    assert torch.isnan(o2[3, :G]).all() and torch.equal(o2[:3], o[:3])
    assert all(bool(torch.isnan(out[p, 0, r])) for p, r in rows[3])
    assert all(torch.equal(out[p, :, r], good[p, :, r]) for b in range(3) for p, r in rows[b])
    assert all(torch.equal(out[p, 1:, r], good[p, 1:, r]) for p, r in rows[3])


# ---------------------------------------------------------------------------- slack
@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=GPU)])
@pytest.mark.parametrize("H,D,page,dtype,lengths,budget,slack", [
    (2, 64, 16, BF, [100, 0, 50, 51, 58, 59, 1], 50, 8), (1, 8, 7, FL, [60, 20, 13, 14], 1, 13),
    (2, 16, 33, FL, [1500, 1100, 1024, 1025], 700, 324), (1, 8, 128, BF, [2500, 3000], 2048, 2 ** 30),
    (2, 8, 64, FL, [20000, 18000, 17999, 5, 300], 17000, 999),        # rows shared out
])
def test_evict_with_slack(dev, H, D, page, dtype, lengths, budget, slack):
    """Rows of up to budget + slack slots keep them all, and their scores and positions go to the new pools as well."""
    _, k, v, table, n = make(len(lengths), H, 1, D, page, lengths, dtype, dev, junk=2.0)
    g = torch.Generator().manual_seed(5)
    scores = torch.rand(k.shape[:3], generator=g).to(dev)
    positions = torch.randint(0, 10 ** 6, k.shape[:3], generator=g, dtype=torch.int32).to(dev)
    seen = torch.full_like(n, 10 ** 6)
    cut = [b for b, m in enumerate(lengths) if m > budget + slack]
    kept = [min(m, budget) if b in cut else m for b, m in enumerate(lengths)]
    want = evict_by_definition((k, v, scores, positions), table[cut], [lengths[b] for b in cut], [10 ** 6] * len(cut), budget, 0)
    k2, v2 = k.clone(), v.clone()
    so, po = torch.full_like(scores, -5.0), torch.full_like(positions, -5)
    got = paged_evict(k2, v2, scores, positions, table, n, seen, budget, scores_out=so, positions_out=po, slack=slack)
    assert got.tolist() == kept
    assert torch.equal(k2, want[0]) and torch.equal(v2, want[1])
    used = torch.zeros(k.shape[:3], dtype=torch.bool)
    for b, m in enumerate(kept):
        s = torch.arange(m)
        used[table.cpu()[b, s // page].long(), :, s % page] = True
    used = used.to(dev)
    assert torch.equal(so[used], want[2][used]) and torch.equal(po[used], want[3][used])
    assert (so[~used] == -5.0).all() and (po[~used] == -5).all()
    assert paged_evict(k, v, scores, positions, table, n, seen, budget, slack=slack).tolist() == kept
    for x, y in zip((k, v, scores, positions), want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=GPU)])
def test_slack_refusals(dev):
    _, k, v, table, n = make(2, 2, 2, 16, 8, [9, 5], BF, dev)
    s, p = torch.zeros(k.shape[:3]).to(dev), torch.zeros(k.shape[:3]).int().to(dev)
    with pytest.raises(RuntimeError, match="slack"):
        paged_evict(k, v, s, p, table, n, n, 4, slack=-1)


# ---------------------------------------------------------------------------- what is written
@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=GPU)])
def test_written_pools_that_require_gradients_are_refused(dev):
    q, k, v, table, n = make(2, 2, 2, 16, 8, [9, 5], FL, dev)
    s, p = torch.zeros(k.shape[:3]).to(dev), torch.zeros(k.shape[:3]).int().to(dev)
    x = torch.zeros(2, 1, 2, 16).to(dev)
    leaf = torch.zeros_like(s).requires_grad_()
    for call in (lambda: paged_attention(q, k, v, table, n, scores=s, scores_out=leaf),
                 lambda: paged_append(x, x, k, v, table, n, scores=leaf),
                 lambda: paged_evict(k, v, s, p, table, n, n, 4, scores_out=leaf)):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
    with torch.no_grad():
        paged_attention(q, k, v, table, n, scores=s, scores_out=leaf)
    assert leaf.detach().any()


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=GPU)])
def test_pools_in_one_place_are_refused(dev):
    """Keys and values, or scores and where they go, that are the same memory in views which are not dense or are laid
    out in another order. Views that lie side by side in one tensor are fine."""
    q, k, v, table, n = make(2, 2, 2, 16, 8, [9, 5], FL, dev, junk=0.0)
    P = k.shape[0]
    s, p = torch.zeros(P, 2, 8).to(dev), torch.zeros(P, 2, 8).int().to(dev)
    x = torch.ones(2, 1, 2, 16).to(dev)
    layers = torch.zeros(P, 4, 8, 16).to(dev)
    one = layers[:, 1:3]
    for call in (lambda: paged_append(x, x, one, layers[:, 1:3], table, n),
                 lambda: paged_evict(one, layers[:, 1:3], s, p, table, n, n, 4)):
        with pytest.raises(RuntimeError):
            call()
    square = torch.rand(P, 8, 8).to(dev)          # 8 heads, pages of 8: the transposed view has the same sizes
    k8, v8 = (torch.zeros(P, 8, 8, 16).to(dev) for _ in range(2))
    p8 = torch.zeros(P, 8, 8).int().to(dev)
    q8 = torch.zeros(2, 8, 16).to(dev)
    for call in (lambda: paged_attention(q8, k8, v8, table, n, scores=square, scores_out=square.transpose(1, 2)),
                 lambda: paged_evict(k8, v8, square, p8, table, n, n, 4, scores_out=square.transpose(1, 2)),
                 lambda: paged_evict(k8, v8, square, p8, table, n, n, 4, positions_out=p8.transpose(1, 2))):
        with pytest.raises(RuntimeError):
            call()
    assert not layers.any()
    paged_append(x, x, layers[:, :2], layers[:, 2:], table, n)
    assert layers.any()
    both = torch.zeros(P, 2, 2, 8).to(dev)
    paged_attention(q, k, v, table, n, scores=both[:, 0], scores_out=both[:, 1])
    paged_attention(q, k, v, table, n, scores=both[:, 0], scores_out=both[:, 0])
    assert both[:, 0].any()


@GPU
@pytest.mark.parametrize("D,H,G,page,dtype,rows,longest,weights", [
    (128, 16, 1, 7, BF, 1400, 40, False), (128, 16, 1, 100, HF, 56, 1000, False),
    (64, 16, 1, 100, BF, 120, 900, True), (64, 16, 2, 7, HF, 62, 1700, False),
    (256, 16, 1, 16, BF, 110, 250, False), (256, 16, 1, 33, HF, 27, 1000, True),
    (128, 16, 1, 64, HF, 130, 400, True), (64, 16, 3, 64, BF, 62, 1700, True), (256, 16, 2, 64, HF, 27, 1000, False),
    (128, 4, 17, 16, BF, 210, 1000, False), (128, 4, 32, 5, HF, 210, 1000, False), (64, 4, 20, 16, BF, 420, 1000, True),
    (256, 4, 17, 100, BF, 110, 1000, False), (128, 16, 1, 7, FL, 56, 500, False), (64, 16, 1, 20, FL, 56, 900, True),
])
def test_16_bits_streamed_past_the_caches(gpu, D, H, G, page, dtype, rows, longest, weights):
    """Every form that takes its keys and values past the caches: head widths, pages of a multiple of 16 rows or of any size,
    one work item to a sequence or several, one or two blocks of query heads, weights gathered or not."""
    lengths = [longest - i % 7 for i in range(rows)]
    assert 2 * H * D * torch.finfo(dtype).bits // 8 * sum(lengths) > 4e8
    width = -(-longest // page)
    g = torch.Generator("cuda").manual_seed(3)
    k, v = (torch.randn(rows * width, H, page, D, generator=g, device="cuda", dtype=dtype) for _ in range(2))
    table = torch.arange(rows * width, dtype=torch.int32, device="cuda").view(width, rows).t().contiguous()
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = torch.randn(rows, H * G, D, generator=g, device="cuda", dtype=dtype)
    s = torch.zeros(k.shape[:3], device="cuda") if weights else None
    o = paged_attention(q, k, v, table, n, scores=s)
    for b in (0, rows // 2, rows - 1):
        m = lengths[b]
        own = table[b].long()
        kb, vb = (t[own].transpose(0, 1).reshape(H, -1, D)[:, :m].double().cpu() for t in (k, v))
        w = torch.softmax(q[b].double().cpu().view(H, G, D) @ kb.transpose(1, 2) / math.sqrt(D), -1)
        close(o[b], (w @ vb).view(H * G, D), (w @ vb.abs()).view(H * G, D), D)
        if weights:
            got = s[own].transpose(0, 1).reshape(H, -1).double().cpu()
            assert not got[:, m:].any()
            want = w.sum(1)
            assert ((got[:, :m] - want).abs() <= (2.0 ** -24 * 40 * (D + 3) + 2.0 ** -23) * want).all()


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=GPU)])
def test_more_tokens_than_a_sequence_can_have(dev):
    """A length is below 2^31 after any call that is taken: up to 2^30 slots and fewer than 2^30 tokens."""
    _, k, v, table, n = make(1, 1, 1, 8, 8, [3], BF, dev)
    x = torch.zeros(1, 1, 1, 8, dtype=BF, device=dev).expand(1, 2 ** 30, 1, 8)
    with pytest.raises(RuntimeError, match="too many tokens"):
        paged_append(x, x, k, v, table, n)
    assert n.tolist() == [3]


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=GPU)])
@pytest.mark.parametrize("dtype", [BF, FL])
@pytest.mark.parametrize("scale", [2.0 ** -96, 2.0 ** 110])
@pytest.mark.parametrize("n,width", [(45, None), (700, None), (900, 400)])
def test_values_of_any_size(dev, dtype, scale, n, width):
    """Outputs are as exact for tiny and for huge values: sums of 900 weighted values of 2^-96 stay above 2^-126 by more than
    the 24 bits of their terms' largest, and of 2^110 below 2^128. Terms below 2^-126 are off by 2^-149 each, which is below
    900 2^-149 2^96 < 2^-43 of the scale."""
    q, k, v, table, lens = make(2, 2, 2, 64, 16, [n, 3], FL, dev, junk=0.0, width=width)
    q, k, v = q.to(dtype), k.to(dtype), (v * scale).to(dtype)
    ref, mag, _ = define(q, k, v, table, [n, 3])
    o = paged_attention(q, k, v, table, lens).double().cpu()
    tol = torch.finfo(dtype).eps / 2 * ref.abs() + 2.0 ** -24 * 40 * 67 * mag + 2.0 ** -43 * scale
    assert ((o - ref).abs() <= tol).all(), ((o - ref).abs() / tol).max().item()


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=GPU)])
@pytest.mark.parametrize("dtype", [BF, FL])
@pytest.mark.parametrize("scale", [2.0 ** -96, 2.0 ** 110])
def test_weights_are_kept_to_float32_for_values_of_any_size(dev, dtype, scale):
    """As test_weights_are_kept_to_float32: scaling by a power of two changes no rounding of normal numbers, and what the two
    slots give is above 2^-126 by 2^20 at least (values of 2^-4 of the scale and more) or moves the output by 2^-149, which is
    2^-53 of the scale."""
    q, k, v, table, n = _cancelling("cpu", dtype)
    v = (v.double() * scale).to(dtype)
    ref, mag, _ = define(q, k, v, table, [2] * 64, scale=1.0)
    o = paged_attention(*(t.to(dev) for t in (q, k, v, table, n)), scale=1.0).double().cpu()
    tol = torch.finfo(dtype).eps / 2 * ref.abs() + 2.0 ** -20 * mag + 2.0 ** -50 * scale
    assert ((o - ref).abs() <= tol).all(), ((o - ref).abs() / tol).max().item()


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=GPU)])
@pytest.mark.parametrize("dtype,least", [(BF, -50.0), (HF, -25.0), (FL, -80.0)])
def test_infinite_values_with_little_weight(dev, dtype, least):
    """An infinite value comes through whatever the bits of its weight, down to exp(least): every part of a weight that is
    split is above 0. With a weight of 0 it is NaN, as 0 times infinity is."""
    g = torch.Generator().manual_seed(3)
    q, k, v, table, n = make(64, 4, 1, 64, 16, [2] * 64, FL, "cpu", seed=1)
    q.zero_()
    q[:, :, 0] = 1.0
    a = torch.rand(64, 4, generator=g) * least
    a[0, 0] = -1000.0
    for b in range(64):
        p = int(table[b, 0])
        k[p, :, :2] = 0.0
        k[p, :, 1, 0] = a[b]
        v[p, :, 1] = math.inf
        v[p, 2:, 1] = -math.inf
    o = paged_attention(*(t.to(dtype).to(dev) for t in (q, k, v)), table.to(dev), n.to(dev), scale=1.0).float().cpu()
    assert torch.isnan(o[0, 0]).all()
    o[0, 0] = math.inf
    assert (o[:, :2] == math.inf).all() and (o[:, 2:] == -math.inf).all()
