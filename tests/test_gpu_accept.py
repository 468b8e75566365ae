"""GPU tests of the walk that keeps the drafted tokens which the samples confirm, and of a whole round of drafted decoding.  Whole numbers and
copied rows: everything has to be equal, what is not named unchanged."""
import random

import pytest
import torch

import qb200
from drafted_ref import F64, attention, dequantized, line_of, tolerance, walk
from test_gpu_tree_attention import BF16, I32, ints, make_pool, make_table, make_tree

pytestmark = pytest.mark.gpu


def drafted(T, counts, seed, agree=0.8):
    """Trees, tokens (few of them, so that siblings repeat one another) and samples that often are a child's token."""
    rng = random.Random(seed)
    trees, tokens, sampled = [], [], []
    for i, c in enumerate(counts):
        n = max(0, min(c, T))
        tree = make_tree(n, T, seed * 100 + i)
        tok = [rng.randrange(5) for _ in range(T)]
        out = []
        for t in range(T):
            children = [j for j in range(t + 1, n) if tree[j] == t]
            out.append(tok[rng.choice(children)] if children and rng.random() < agree else rng.randrange(5))
        trees.append(tree)
        tokens.append(tok)
        sampled.append(out)
    return trees, tokens, sampled


def expected(pools, table, lens, page, trees, tokens, sampled, counts, rows, T):
    pools = [p.clone() for p in pools]
    path, nxt, acc, ends, done = [], [], [], [], set()
    for b in range(len(trees)):
        r = b if rows is None else rows[b]
        length = max(0, min(lens[r], len(table[r]) * page)) if 0 <= r < len(table) else 0
        n = 0 if r in done else max(0, min(counts[b], T, length))
        done.add(r)
        w = walk(trees[b], tokens[b], sampled[b], n)
        base = length - n
        path.append(w + [-1] * (T - len(w)))
        nxt.append([sampled[b][t] for t in w] + [-1] * (T - len(w)))
        acc.append(len(w))
        ends.append(base + len(w))
        for p in pools:
            before = p.clone() if w else None
            for i, t in enumerate(w):
                to, frm = table[r][(base + i) // page], table[r][(base + t) // page]
                if 0 <= to < p.shape[0] and 0 <= frm < p.shape[0]:
                    p[to, :, (base + i) % page] = before[frm, :, (base + t) % page]
    return pools, path, nxt, acc, ends


def check(pools, table, lens, page, T, counts, seed, rows=None, agree=0.8, give_counts=True):
    trees, tokens, sampled = drafted(T, counts, seed, agree)
    want = expected(pools, table, lens, page, trees, tokens, sampled, counts, rows, T)
    path, nxt, acc, ends = qb200.kv_pages_accept(pools, ints(table), ints(lens), page, ints(trees), ints(tokens), ints(sampled),
                                                 rows=None if rows is None else ints(rows), counts=ints(counts) if give_counts else None)
    assert path.tolist() == want[1]
    assert nxt.tolist() == want[2]
    assert acc.tolist() == want[3]
    assert ends.tolist() == want[4]
    for i, (p, w) in enumerate(zip(pools, want[0])):
        assert torch.equal(p, w), f"pool {i}"
    return want[3]


def tensors(pool):
    return [t for t in pool if t is not None]


@pytest.mark.parametrize("bits,D", [(4, 64), (4, 128), (8, 128), (16, 64), (16, 128), (4, 192)])
@pytest.mark.parametrize("page", [16, 64])
def test_walks_and_rows(bits, D, page):
    torch.manual_seed(1)
    lens = [40, 100, 33, 64, 5, 130]
    pools = [t for _ in range(4) for t in tensors(make_pool(40, 3, page, D, bits))]
    table = make_table(lens, page, 12, 40)
    for seed in range(3):
        n = check(pools, table, lens, page, 33, [1, 12, 33, 20, 5, 7], seed)
    assert max(n) > 2
    check(pools, table, lens, page, 64, [1, 64, 33, 64, 5, 63], 9, agree=0.95)


def test_ends_of_counts_and_wrong_entries():
    torch.manual_seed(2)
    page, lens = 16, [40, 0, 3, 50, 30]
    pools = tensors(make_pool(20, 2, page, 64, 4)) + tensors(make_pool(20, 1, page, 128, 16))
    table = make_table(lens, page, 4, 20)
    check(pools, table, lens, page, 8, [0, 4, 8, 100, -7], 3)
    check(pools, table, lens, page, 8, [8, 8, 8, 8, 8], 4, rows=[4, 3, 4, -1, 99], agree=1.0)   # a sequence listed again, two that do not exist
    table[0][2], table[3][3] = -1, 1000
    check(pools, table, lens, page, 20, [20, 20, 20, 20, 20], 5, give_counts=False)
    check([], table, lens, page, 20, [20, 20, 20, 20, 20], 6)
    check(pools, table, [100, 10 ** 6, -4, 50, 30], page, 8, [8] * 5, 7)                        # lengths beyond the table


def test_chains_and_full_paths():
    """Everything accepted: nothing moves.  Nothing but the root: one token."""
    torch.manual_seed(3)
    page, lens, T = 32, [70, 64], 64
    pools = tensors(make_pool(8, 2, page, 128, 8))
    table = make_table(lens, page, 3, 8)
    before = [p.clone() for p in pools]
    chain, tok = ints([[i - 1 for i in range(T)]] * 2), ints([[100 + i for i in range(T)]] * 2)
    good = ints([[101 + i for i in range(T)]] * 2)
    path, nxt, acc, ends = qb200.kv_pages_accept(pools, ints(table), ints(lens), page, chain, tok, good)
    assert acc.tolist() == [64, 64] and ends.tolist() == lens and torch.equal(nxt, good) and path.tolist() == [list(range(T))] * 2
    path, nxt, acc, ends = qb200.kv_pages_accept(pools, ints(table), ints(lens), page, chain, tok, ints([[7] * T] * 2))
    assert acc.tolist() == [1, 1] and ends.tolist() == [7, 1] and nxt[:, 0].tolist() == [7, 7]
    assert all(torch.equal(a, b) for a, b in zip(pools, before))


def test_pools_of_many_layers_layouts_and_types():
    torch.manual_seed(4)
    page, lens, P = 16, [60, 44], 12
    table = make_table(lens, page, 5, P)
    many = torch.randint(0, 2 ** 31 - 1, (130, P, 2, page, 8), dtype=I32, device="cuda")       # more than one launch takes
    check(list(many.unbind(0)), table, lens, page, 24, [24, 17], 5)
    odd = [torch.randint(0, 255, (P, 3, page, 7), device="cuda").to(torch.uint8), torch.randn(P, 1, page, 5, device="cuda").half(),
           torch.randn(P, 2, page, 33, device="cuda"), torch.randn(P, page, 2, 24, device="cuda").to(BF16).transpose(1, 2),
           torch.randn(P, 2, page, 40, device="cuda").to(BF16)[..., 3:35], torch.randn(2, P, page, 16, device="cuda").transpose(0, 1)]
    check(odd, table, lens, page, 24, [24, 24], 6)
    # what lies between the rows stays
    base = torch.randn(P, 2, page, 40, device="cuda")
    keep = base.clone()
    check([base[..., 4:36]], table, lens, page, 24, [24, 24], 7)
    assert torch.equal(base[..., :4], keep[..., :4]) and torch.equal(base[..., 36:], keep[..., 36:])


def test_many_sequences_lists_with_strides_streams_and_graphs():
    torch.manual_seed(5)
    page, B, T = 16, 150, 11
    lens = [T + (13 * i) % 90 for i in range(B)]
    P = sum(-(-n // page) for n in lens) + 1
    pools = tensors(make_pool(P, 1, page, 64, 4))
    table = make_table(lens, page, 8, P)
    check(pools, table, lens, page, T, [1 + i % T for i in range(B)], 8)
    trees, tokens, sampled = drafted(T, [T] * B, 9)
    wide = torch.full((3, B, T + 5), 2, dtype=I32, device="cuda")
    for i, x in enumerate((trees, tokens, sampled)):
        wide[i, :, 1:T + 1] = ints(x)
    lists = [wide[i, :, 1:T + 1] for i in range(3)]
    copies = [p.clone() for p in pools]
    graph = torch.cuda.CUDAGraph()
    dt, dl = ints(table), ints(lens)
    with torch.cuda.graph(graph):
        got = qb200.kv_pages_accept(copies, dt, dl, page, *lists)
    for c, p in zip(copies, pools):
        c.copy_(p)
    graph.replay()
    torch.cuda.synchronize()
    want = expected(pools, table, lens, page, trees, tokens, sampled, [T] * B, None, T)
    assert [x.tolist() for x in got] == list(want[1:])
    assert all(torch.equal(a, b) for a, b in zip(copies, want[0]))


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_rounds_of_drafted_decoding(bits):
    """Three rounds for three sequences, two of them answers of one prompt: reserve, append, attention of the trees, sampling, the walk, and
    the rest given back.  The caches afterwards are those of the confirmed tokens alone, and the samples those of their own attention."""
    torch.manual_seed(6)
    page, Hkv, Hq, D, T, layers, P, S, V = 16, 2, 8, 64, 9, 2, 64, 3, 50
    scale = D ** -0.5
    caches = [[make_pool(P, Hkv, page, D, bits) for _ in range(2)] for _ in range(layers)]
    pools = [t for layer in caches for side in layer for t in tensors(side)]
    table, lens, refs = torch.full((S, 8), -1, dtype=I32, device="cuda"), torch.zeros(S, dtype=I32, device="cuda"), torch.zeros(P, dtype=I32, device="cuda")
    # a token's key, value and query are made from its number and its place on its line; its logits from the attention
    embed = torch.randn(V, layers, Hkv * 2 + Hq, D, device="cuda")
    head = torch.randn(Hq * D, V, device="cuda")

    def rows_of(token, position, layer):
        x = embed[token, layer] * torch.cos(0.1 * position + torch.arange(D, device="cuda"))
        return x.to(BF16)

    def dense(tokens, positions, layer):
        x = torch.stack([rows_of(t, p, layer) for t, p in zip(tokens, positions)])             # [n, heads, D]
        return x[:, :Hkv].transpose(0, 1), x[:, Hkv:2 * Hkv].transpose(0, 1), x[:, 2 * Hkv:].transpose(0, 1)

    texts = [[random.Random(1).randrange(V) for _ in range(37)], None, [random.Random(2).randrange(V) for _ in range(16)]]
    for s in (0, 2):
        n = len(texts[s])
        pos, pairs = qb200.kv_pages_reserve(table, lens, refs, page, ints([s]), ints([n]))
        for layer in range(layers):
            k, v, _ = dense(texts[s], range(n), layer)
            qb200.kv_pages_append(*caches[layer], k[None].contiguous(), v[None].contiguous(), table, pos, bits, 64, rows=ints([s]))
    assert qb200.kv_pages_fork(table, lens, refs, page, ints([0]), ints([1])).tolist() == [37]
    texts[1] = list(texts[0])
    certain = [3, 4, 5]                                   # the last token of each, not yet in the cache
    total = 0
    for turn in range(3):
        trees, tokens, counts = [], [], [T, T - 2, T]
        for s in range(S):
            tree = make_tree(counts[s], T, 50 * turn + s)
            trees.append([-1] + [0 if p < 0 else p for p in tree[1:]])
            rng = random.Random(turn * 10 + s)
            tokens.append([certain[s]] + [rng.randrange(V) for _ in range(T - 1)])
        pos, pairs = qb200.kv_pages_reserve(table, lens, refs, page, ints([0, 1, 2]), ints(counts))
        qb200.kv_pages_copy(pools, pairs)
        base = [len(t) for t in texts]
        assert pos.tolist() == base
        depth = [[len(line_of(trees[s][:counts[s]] + [-1] * T, t)) - 1 for t in range(T)] for s in range(S)]
        hidden = torch.zeros(S, T, Hq * D, device="cuda")
        for layer in range(layers):
            kvq = [dense(tokens[s], [base[s] + d for d in depth[s]], layer) for s in range(S)]
            k, v, q = (torch.stack([x[i] for x in kvq]).contiguous() for i in range(3))
            qb200.kv_pages_append(*caches[layer], k, v, table, pos, bits, 64, rows=ints([0, 1, 2]), counts=ints(counts))
            out = qb200.kv_pages_tree_attention(q, *caches[layer], table, lens, ints(trees), bits, 64, scale, counts=ints(counts))
            hidden += out.float().transpose(1, 2).reshape(S, T, Hq * D)
        logits = (hidden @ head).reshape(S * T, V)
        # the drafts are made to agree with the samples along one line, as a good drafter's would
        u = torch.rand(S * T, device="cuda")
        sampled = qb200.sample(logits, u, torch.full((S * T,), 0.8, device="cuda"), torch.full((S * T,), 20, dtype=I32, device="cuda")).reshape(S, T)
        chosen, draft = sampled.tolist(), [list(t) for t in tokens]
        for s in range(S):
            at = 0
            for child in range(1, counts[s]):
                if trees[s][child] == at and child % 2:
                    chosen[s][at] = draft[s][child]
                    at = child
        path, nxt, acc, ends = qb200.kv_pages_accept(pools, table, lens, page, ints(trees), ints(draft), ints(chosen), counts=ints(counts))
        qb200.kv_pages_free(table, lens, refs, page, ints([0, 1, 2]), begin=ends)
        for s in range(S):
            w = walk(trees[s], draft[s], chosen[s], counts[s])
            assert path.tolist()[s][: len(w)] == w and acc.tolist()[s] == len(w)
            texts[s] += [draft[s][t] for t in w]
            certain[s] = chosen[s][w[-1]]
            assert nxt.tolist()[s][len(w) - 1] == certain[s]
            total += len(w)
        assert lens.tolist() == [len(t) for t in texts] == ends.tolist()
        # every cached row is the row of its token at its position, quantised as an append would
        rows = table.tolist()
        for s in range(S):
            used = [rows[s][p] for p in range(-(-len(texts[s]) // page))]
            assert all(e >= 0 for e in used) and all(e < 0 for e in rows[s][len(used):])
            for layer in range(layers):
                k, v, _ = dense(texts[s], range(len(texts[s])), layer)
                for side, want in zip(caches[layer], (k, v)):
                    for got, ref in zip(tensors(side), [want.contiguous()] if bits == 16 else qb200.quantize(want.contiguous(), 64, bits)):
                        at = torch.arange(len(texts[s]), device="cuda")
                        mine = got[torch.tensor(used, device="cuda")[at // page], :, at % page].transpose(0, 1)
                        assert torch.equal(mine, ref)
    assert total > 12
    live = set(e for r in table.tolist() for e in r if e >= 0)
    assert {i for i, c in enumerate(refs.tolist()) if c > 0} == live
    # and the next token's attention over what is there now
    q = torch.randn(S, Hq, 1, D, device="cuda").to(BF16)
    out = qb200.kv_pages_tree_attention(q, *caches[0], table, lens, ints([[-1]] * S), bits, 64, scale)
    kd, vd = dequantized(caches[0][0], bits), dequantized(caches[0][1], bits)
    for s in range(S):
        at = torch.arange(len(texts[s]), device="cuda")
        pid = table[s][(at // page)].long()
        for h in range(Hkv):
            o, A, sc = attention(q[s, h * 4:(h + 1) * 4, 0].to(F64), kd[pid, h, at % page], vd[pid, h, at % page], scale)
            assert ((out[s, h * 4:(h + 1) * 4, 0].to(F64) - o).abs() <= tolerance(o, A, sc, bits, vd[pid, h, at % page])).all()
