"""GPU tests of the paged cache: rows into pages, the bookkeeping against its rules step by step, page copies."""
import random

import pytest
import torch

import qb200
from pages_ref import State

pytestmark = pytest.mark.gpu
I32, BF16 = torch.int32, torch.bfloat16


def ints(x):
    return torch.tensor(x, dtype=I32, device="cuda")


def make_pool(P, H, page, D, bits, fill=None):
    """Pool of noise, so that rows that change without being asked to are seen."""
    if bits == 16:
        return (torch.randn(P, H, page, D, device="cuda").to(BF16), None, None)
    return (torch.randint(-2 ** 31, 2 ** 31 - 1, (P, H, page, D * bits // 32), device="cuda", dtype=torch.int64).to(I32),
            torch.randn(P, H, page, D // 64, device="cuda").to(BF16), torch.randn(P, H, page, D // 64, device="cuda").to(BF16))


def tensors(pool):
    return [t for t in pool if t is not None]


def permuted(pool):
    """The same pool with the head axis innermost of the page: [pages, page, heads, cols] in memory."""
    return tuple(None if t is None else t.transpose(1, 2).contiguous().transpose(1, 2) for t in pool)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("D,page,H,S,layout", [(128, 16, 3, 1, "plain"), (64, 32, 1, 37, "plain"), (128, 64, 2, 70, "heads"), (192, 16, 2, 19, "dense"), (64, 128, 5, 130, "heads")])
def test_append_writes_its_rows_and_no_others(bits, D, page, H, S, layout):
    torch.manual_seed(bits + D + S)
    N, M, P, seqs = 5, 4 + (S + page) // page, 60, 7
    kp, vp = make_pool(P, H, page, D, bits), make_pool(P, H, page, D, bits)
    if layout == "heads":
        kp, vp = permuted(kp), permuted(vp)
    if layout == "dense":       # rows that start off 16 bytes, a head stride of its own
        dk, dv = (torch.randn(N, H, S + 2, D + 3, device="cuda").to(BF16)[:, :, 1:S + 1, 1:D + 1] for _ in range(2))
    else:
        dk, dv = (torch.randn(N, H, S, D, device="cuda").to(BF16) for _ in range(2))
    perm = torch.randperm(P)[:seqs * M].tolist() if seqs * M <= P else [i % P for i in range(seqs * M)]
    table = [perm[i * M:(i + 1) * M] for i in range(seqs)]
    if seqs * M > P:            # every sequence written to has pages of its own
        free = list(range(P))
        random.Random(S).shuffle(free)
        table = [[free.pop() if free else -1 for _ in range(M)] for _ in range(seqs)]
    table[2][0], table[4][1] = -1, P            # no page, a number outside the pool
    rows, pos = [3, 2, 4, 9, -1], [0, page - 1, 7, 0, 0]
    counts = [S, S, max(1, S - 3), S, S]
    want_k, want_v = ([None if t is None else t.clone() for t in p] for p in (kp, vp))
    for n in range(N):
        for i in range(min(S, counts[n])):
            r, at = rows[n], pos[n] + i
            if not 0 <= r < seqs or at // page >= M or not 0 <= table[r][at // page] < P:
                continue
            for want, dense in ((want_k, dk), (want_v, dv)):
                x = dense[n, :, i].contiguous()
                new = (x,) if bits == 16 else qb200.quantize(x, 64, bits)
                for t, v in zip(want, new):
                    t[table[r][at // page], :, at % page] = v
    qb200.kv_pages_append(kp, vp, dk, dv, ints(table), ints(pos), bits, 64, rows=ints(rows), counts=ints(counts))
    for got, want in zip(tensors(kp) + tensors(vp), tensors(want_k) + tensors(want_v)):
        assert torch.equal(got.view(torch.int16) if got.dtype == BF16 else got, want.view(torch.int16) if want.dtype == BF16 else want)


def test_append_drops_positions_below_zero_and_counts_of_none():
    kp, vp = make_pool(4, 2, 16, 64, 4), make_pool(4, 2, 16, 64, 4)
    before = [t.clone() for t in tensors(kp) + tensors(vp)]
    x = torch.randn(2, 2, 3, 64, device="cuda").to(BF16)
    qb200.kv_pages_append(kp, vp, x, x, ints([[0], [1]]), ints([-3, 5]), 4, counts=ints([3, 0]))
    assert all(torch.equal(a, b) for a, b in zip(before, tensors(kp) + tensors(vp)))
    qb200.kv_pages_append(kp, vp, x, x, ints([[0], [1]]), ints([-1, 2 ** 31 - 2]), 4)     # only tokens 1 and 2 of the first have places
    want = qb200.quantize(x[0, :, 1:].contiguous(), 64, 4)[0]
    assert torch.equal(kp[0][0, :, :2], want) and torch.equal(kp[0][1:], before[0][1:])


@pytest.mark.parametrize("bits", [4, 8])
def test_codes_are_those_of_a_division(bits):
    """Groups whose quotients are ties, or next to one, as often as bf16 values make them so, at every magnitude; the codes by a division
    in fp32 rounded to nearest even, worked out here."""
    g = torch.Generator(device="cuda").manual_seed(bits)
    rows = 4096
    x = torch.randint(-255, 256, (rows, 64), device="cuda", generator=g).float() * 2.0 ** torch.randint(-30, 30, (rows, 1), device="cuda", generator=g).float()
    x[::2] = torch.randn(rows // 2, 64, device="cuda", generator=g) * 2.0 ** torch.randint(-40, 100, (rows // 2, 1), device="cuda", generator=g).float()
    x[:64] = torch.arange(64, device="cuda") * torch.arange(1, 65, device="cuda")[:, None] / 2.0
    x = x.to(BF16)
    v = x.float()
    lo, hi = v.amin(1, keepdim=True), v.amax(1, keepdim=True)
    bins = torch.full_like(lo, 2.0 ** bits - 1)
    neg = lo.abs() > hi.abs()
    s = torch.clamp((hi - lo) / bins, min=1e-7)
    s = torch.where(neg, s, -s)
    edge = torch.where(neg, lo, hi)
    q0 = torch.round(edge / s)
    s = torch.where(q0 == 0, s, edge / torch.where(q0 == 0, torch.ones_like(q0), q0))
    bias = torch.where(q0 == 0, torch.zeros_like(edge), edge)
    want = torch.minimum(torch.clamp(torch.round((v - bias) / s), min=0.0), bins).to(torch.int64)
    q, sc, b = qb200.quantize(x, 64, bits)
    got = ((q[..., None].to(torch.int64) >> (torch.arange(32 // bits, device="cuda") * bits)) & (2 ** bits - 1)).reshape(rows, 64)
    assert torch.equal(got, want) and torch.equal(sc, s.to(BF16)) and torch.equal(b, bias.to(BF16))


# ---------------------------------------------------------------- bookkeeping

class Both:
    """The device's state beside the restated one."""

    def __init__(self, S, M, P, page):
        self.ref = State(S, M, P, page)
        wide = torch.full((S, M + 3), -7, dtype=I32, device="cuda")
        wide[:, :M] = -1
        self.wide, self.table = wide, wide[:, :M]           # a table with a row stride of its own
        self.lens, self.refs, self.page = ints([0] * S), ints([0] * P), page

    def check(self):
        assert self.table.tolist() == self.ref.table and self.lens.tolist() == self.ref.lens and self.refs.tolist() == self.ref.refs
        assert bool((self.wide[:, self.ref.M:] == -7).all())
        used = [0] * self.ref.P                             # what the counts stand for
        for row in self.ref.table:
            for e in row:
                if e >= 0:
                    used[e] += 1
        assert used == self.ref.refs

    def reserve(self, rows, counts):
        pos, copies = qb200.kv_pages_reserve(self.table, self.lens, self.refs, self.page, ints(rows), ints(counts))
        wp, wc = self.ref.reserve(rows, counts)
        assert pos.tolist() == wp and [tuple(c) for c in copies.tolist()] == wc
        self.check()
        return wp, wc

    def fork(self, src, dst, tokens=None):
        got = qb200.kv_pages_fork(self.table, self.lens, self.refs, self.page, ints(src), ints(dst), None if tokens is None else ints(tokens))
        want = self.ref.fork(src, dst, tokens)
        assert got.tolist() == want
        self.check()
        return want

    def free(self, rows, begin=None, end=None):
        qb200.kv_pages_free(self.table, self.lens, self.refs, self.page, ints(rows), None if begin is None else ints(begin), None if end is None else ints(end))
        self.ref.free(rows, begin, end)
        self.check()

    def compact(self):
        remap, moves, count = qb200.kv_pages_compact(self.table, self.refs)
        wr, wm = self.ref.compact()
        assert remap.tolist() == wr and count.item() == len(wm)
        assert [tuple(m) for m in moves.tolist()] == wm + [(-1, -1)] * (self.ref.P // 2 - len(wm))
        self.check()


@pytest.mark.parametrize("S,M,P,page", [(1, 1, 1, 16), (6, 5, 17, 16), (9, 12, 64, 32), (30, 40, 700, 64), (12, 7, 33, 16)])
@pytest.mark.parametrize("clusters", [True, False])
def test_bookkeeping_step_by_step(S, M, P, page, clusters, request):
    if not clusters:
        request.getfixturevalue("no_clusters")
    rng = random.Random(S * 1000 + P)
    st = Both(S, M, P, page)
    pick = lambda: rng.randint(-1, S)
    for _ in range(40):
        op = rng.choice(["reserve", "reserve", "fork", "free", "compact", "window"])
        n = rng.randint(1, S + 2)
        if op == "reserve":
            st.reserve([pick() for _ in range(n)], [rng.choice([0, 1, 1, page, rng.randint(-1, 3 * page)]) for _ in range(n)])
        elif op == "fork":
            st.fork([pick() for _ in range(n)], [pick() for _ in range(n)], rng.choice([None, [rng.randint(-2, M * page) for _ in range(n)]]))
        elif op == "free":
            st.free([pick() for _ in range(n)], rng.choice([None, [rng.randint(-5, M * page) for _ in range(n)]]))
        elif op == "window":
            st.free([pick() for _ in range(n)], [rng.choice([0, 4, page]) for _ in range(n)], [rng.randint(0, M * page) for _ in range(n)])
        else:
            st.compact()


def test_a_pool_that_runs_out_serves_the_list_up_to_there():
    st = Both(5, 4, 6, 16)
    pos, _ = st.reserve([0, 1, 2, 3], [40, 17, 33, 0])
    assert pos == [0, 0, -1, 0]
    assert st.reserve([2, 1], [17, 15])[0] == [-1, 17]     # the second one needs no page
    st.free([0])
    assert st.reserve([2], [17])[0] == [0]


def test_reserve_of_a_large_pool_and_long_lists():
    """More pages than one pass of a block, fresh pages across the blocks' shares."""
    st = Both(300, 30, 20000, 16)
    st.reserve(list(range(300)), [(7 * i) % 480 + 1 for i in range(300)])
    st.free([i for i in range(300) if i % 3 == 0])
    st.fork([1, 2] * 50, [i for i in range(300) if i % 3 == 0])
    st.reserve([i for i in range(300) if i % 3 == 0], [5] * 100)
    st.free([i for i in range(300) if i % 2])
    st.compact()


# ---------------------------------------------------------------- copies

@pytest.mark.parametrize("shape,dtype,view", [
    ((9, 2, 16, 16), I32, None), ((9, 3, 16, 1), BF16, None), ((9, 5), torch.uint8, None), ((9, 7, 3), torch.float16, None), ((9, 2, 16, 64), BF16, "heads"),
    ((9, 4, 32, 8), I32, "part"), ((9, 4, 32, 7), BF16, "part"), ((9, 4096, 5), torch.float32, None), ((9, 1), BF16, None), ((9, 33, 5), torch.int8, "part")])
def test_copy_moves_whole_pages(shape, dtype, view):
    g = torch.Generator(device="cuda").manual_seed(len(shape))
    make = lambda s: torch.randint(0, 100, s, device="cuda", generator=g).to(dtype)
    if view == "heads":
        x = make((shape[0], shape[2], shape[1], shape[3])).transpose(1, 2)
    elif view == "part":
        x = make(tuple(s + (2 if i else 0) for i, s in enumerate(shape)))[tuple(slice(0, s) for s in shape)]
    else:
        x = make(shape)
    other = make((9, 3))
    base = x._base.clone() if x._base is not None else x.clone()
    want, want_other = x.clone(), other.clone()
    pairs = [(0, 5), (-1, -1), (3, 1), (9, 2), (4, 9), (7, 7), (8, -3), (2, 6)]
    for s, d in [(0, 5), (3, 1), (2, 6)]:
        want[d], want_other[d] = x[s], other[s]
    qb200.kv_pages_copy([x, other], ints(pairs))
    assert torch.equal(x, want) and torch.equal(other, want_other)
    if view == "part":          # what lies around the pages stays
        now = x._base.clone()
        now[tuple(slice(0, s) for s in shape)] = base[tuple(slice(0, s) for s in shape)]
        assert torch.equal(now, base)


def test_copy_takes_the_count_from_the_device_and_many_pools():
    pools = [torch.arange(8 * 40, device="cuda", dtype=I32).reshape(8, 40) * (i + 1) for i in range(200)]
    want = [p.clone() for p in pools]
    pairs = ints([(0, 4), (1, 5), (2, 6), (3, 7)])
    for n, upto in ((2, 2), (-1, 0), (9, 4)):
        qb200.kv_pages_copy(pools, pairs, ints([n]))
        for w in want:
            w[4:4 + upto] = w[:upto]
        assert all(torch.equal(a, b) for a, b in zip(pools, want))


def test_forks_that_grow_apart():
    """The calls in a row: one prompt, three answers that share it, a token each, the copies, a freed one, a compact pool -- every
    sequence reads back what it wrote."""
    torch.manual_seed(0)
    S, M, P, page, H, D, bits = 5, 6, 24, 16, 2, 64, 4
    st = Both(S, M, P, page)
    kp, vp = make_pool(P, H, page, D, bits), make_pool(P, H, page, D, bits)
    hist = {r: torch.zeros(H, 0, D, device="cuda", dtype=BF16) for r in range(S)}

    def grow(rows, n):
        x = torch.randn(len(rows), H, n, D, device="cuda").to(BF16)
        pos, copies = st.reserve(rows, [n] * len(rows))
        qb200.kv_pages_copy(tensors(kp) + tensors(vp), ints(copies))
        qb200.kv_pages_append(kp, vp, x, -x, st.table, ints(pos), bits, 64, rows=ints(rows))
        for r, v in zip(rows, x):
            hist[r] = torch.cat([hist[r], v], 1)

    def check():
        for r in range(S):
            n = st.ref.lens[r]
            assert n == hist[r].shape[1]
            if n == 0:
                continue
            at = torch.arange(n, device="cuda")
            pid = st.table[r].long()[at // page]
            want = qb200.quantize(hist[r], 64, bits), qb200.quantize(-hist[r], 64, bits)
            for pool, w in zip((kp, vp), want):
                for t, v in zip(pool, w):
                    assert torch.equal(t[pid, :, at % page].transpose(0, 1), v)

    grow([0], 37)
    assert st.fork([0, 0, 0], [1, 2, 3], None) == [37, 37, 37]
    for r in (1, 2, 3):
        hist[r] = hist[0]
    grow([1, 0, 2], 1)
    grow([3, 1], 13)
    check()
    st.free([0, 2], [0, 16])
    hist[0], hist[2] = hist[0][:, :0], hist[2][:, :16]
    grow([2], 1)
    remap, moves, count = qb200.kv_pages_compact(st.table, st.refs)
    st.ref.compact()
    st.check()
    qb200.kv_pages_copy(tensors(kp) + tensors(vp), moves, count)
    check()
    assert max(max(row) for row in st.ref.table) + 1 == sum(r > 0 for r in st.ref.refs)


def test_bookkeeping_in_a_replayed_graph():
    """Fork, reserve and free in one captured graph, replayed on a state that changed in between."""
    st = Both(6, 8, 40, 16)
    st.reserve([0, 1], [30, 16])
    src, dst, ones = ints([0, 1, 0]), ints([2, 3, 4]), ints([1, 1, 1])
    args = (st.table, st.lens, st.refs, 16)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            shared = qb200.kv_pages_fork(*args, src, dst)
            pos, copies = qb200.kv_pages_reserve(*args, dst, ones)
            qb200.kv_pages_free(*args, dst)
    for extra in (0, 5, 20):
        st.reserve([0, 1], [extra, extra])
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want = st.ref.fork([0, 1, 0], [2, 3, 4])
        wp, wc = st.ref.reserve([2, 3, 4], [1, 1, 1])
        st.ref.free([2, 3, 4])
        assert shared.tolist() == want and pos.tolist() == wp and [tuple(c) for c in copies.tolist()] == wc
        st.check()


@pytest.mark.parametrize("S,M,P", [(3, 1100, 2000), (700, 513, 100000), (1, 1, 1), (5, 0, 64)])
def test_compact_rewrites_tables_of_any_shape(S, M, P):
    """Rows of several chunks, more rows than one pass of the device takes, with strides, shared and foreign pages among the entries."""
    g = torch.Generator(device="cuda").manual_seed(S)
    wide = torch.full((S, M + 3), -7, dtype=torch.int32, device="cuda")
    table = wide[:, :M]
    table.copy_(torch.randint(-P, P, (S, M), device="cuda", generator=g, dtype=torch.int32))
    if M:
        table[0, 0] = P + 5                                   # no page of the pool: no page behind the call either
    refs = torch.zeros(P, dtype=torch.int32, device="cuda")
    named = table[(table >= 0) & (table < P)].long()
    refs.scatter_add_(0, named, torch.ones_like(named, dtype=torch.int32))
    before, counts = table.clone(), refs.clone()
    remap, moves, count = qb200.kv_pages_compact(table, refs)
    live = int((counts > 0).sum())
    back = torch.nonzero((counts > 0) & (torch.arange(P, device="cuda") >= live)).flatten()
    holes = torch.nonzero((counts == 0) & (torch.arange(P, device="cuda") < live)).flatten()
    want = torch.where(counts > 0, torch.arange(P, device="cuda"), -1)
    want[back] = holes
    assert count.item() == len(back) and torch.equal(remap.long(), want)
    assert torch.equal(moves[:len(back)].long(), torch.stack([back, holes], 1)) and bool((moves[len(back):] == -1).all())
    entries = torch.where((before >= 0) & (before < P), want[before.clamp(0, P - 1).long()], torch.where(before < 0, before, -1).long())
    assert torch.equal(table.long(), entries) and bool((wide[:, M:] == -7).all())
    moved = torch.zeros_like(counts)
    moved[want[counts > 0]] = counts[counts > 0]
    assert torch.equal(refs, moved)
