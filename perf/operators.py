"""The paged key-value cache as cases that can be timed: new rows into pages, the bookkeeping of the pages (fork, reserve,
free, compact, copy), attention of one new token over pages, and attention of a prompt with a sliding window and sinks.

A case is a dict of plain values; ``kind`` picks the operator.  With ``own`` false ``run`` computes in elementary torch
operations in fp32; with ``own`` true it makes the library's calls.  Head layouts and lengths are those of this repository's
benchmark configurations (32 query heads on 8 cache heads of 128, caches of 32k tokens, 16 sequences) and of its tests (7 query
heads to a cache head, head dim 64, odd lengths); page sizes and windows are generic.

Cache pages: a pool is [pages, heads, page, cols]; at 4 and 8 bits a triple of packed codes (int32 words, lowest bits first),
bf16 scales and biases per 64 values, at 16 bits the bf16 rows themselves.  ``table`` [sequences, pages of a sequence] holds page
numbers, -1 where there is none; ``lens`` the tokens of a sequence; ``refs`` how many table entries name a page (0: free).
"""
import math
import os
import sys

import torch

own = False
BF16, I32 = torch.bfloat16, torch.int32
GROUP = 64


def _lib():
    path = os.path.abspath("mlx-serve_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import qb200
    return qb200


# ---------------------------------------------------------------- cases

def listed():
    return [
        # One layer's new rows of a decode tick: 13 users, one token each.  Latency of a launch.
        {"name": "append_tick", "kind": "append", "N": 13, "S": 1, "Hkv": 8, "D": 128, "bits": 4, "page": 64, "M": 64, "pos": 129},
        # Two prompt chunks of up to 4096 tokens into an 8-bit cache, at an odd position, the second one shorter.
        {"name": "append_prompt", "kind": "append", "N": 2, "S": 4096, "Hkv": 8, "D": 128, "bits": 8, "page": 64, "M": 72, "pos": 129},
        # Three more answers of one prompt begin: the sequences of the last answers are freed, the prompt's pages are shared,
        # a slot for the next token is reserved and the half-filled last page is copied, in two layers.
        {"name": "pages_fork_3", "kind": "fork", "parents": 1, "children": 3, "layers": 2, "T": 1000, "Hkv": 8, "D": 128, "bits": 4, "page": 64, "P": 160},
        # The same for eight prompts with seven answers each over sixteen layers: the copies are what takes time.
        {"name": "pages_fork_56", "kind": "fork", "parents": 8, "children": 7, "layers": 16, "T": 2500, "Hkv": 8, "D": 128, "bits": 4, "page": 64, "P": 700},
        # Housekeeping of a server whose layers have a window: pages that left the window are freed, those that stay move
        # to the front of the pool, in eight layers.
        {"name": "pages_compact_24", "kind": "compact", "rows": 24, "layers": 8, "T": 4096, "window": 1024, "sinks": 4, "Hkv": 8, "D": 128, "bits": 8, "page": 32,
         "P": 3200},
        # One user, a short context: the smallest attention call, where the fixed part counts.
        {"name": "decode_1_seq", "kind": "decode", "B": 1, "Hq": 32, "Hkv": 8, "D": 128, "T": 700, "window": 0, "sinks": 0, "bits": 4, "page": 64},
        # Thirteen users of very different lengths, seven query heads to a cache head, 8 bits, small pages.
        {"name": "decode_13_ragged", "kind": "decode", "B": 13, "Hq": 28, "Hkv": 4, "D": 128, "T": 8191, "window": 0, "sinks": 0, "bits": 8, "page": 16},
        # A layer with a window over an unquantised cache: 32 users, each sees four first tokens and the last 1024.
        {"name": "decode_32_window", "kind": "decode", "B": 32, "Hq": 64, "Hkv": 8, "D": 64, "T": 16384, "window": 1024, "sinks": 4, "bits": 16, "page": 128},
        # Sixteen users of up to 32k tokens at 4 bits: the largest read of the cache.
        {"name": "decode_16_32k", "kind": "decode", "B": 16, "Hq": 32, "Hkv": 8, "D": 128, "T": 32768, "window": 0, "sinks": 0, "bits": 4, "page": 64},
        # A short prompt of a small model: one tile, a window inside it.
        {"name": "window_77", "kind": "window", "B": 1, "Hq": 8, "Hkv": 2, "D": 64, "Tq": 77, "Tk": 77, "window": 32, "sinks": 2, "lens": False},
        # A chunk of 512 tokens behind 3587 cached ones (chunked prefill).
        {"name": "window_chunk", "kind": "window", "B": 1, "Hq": 32, "Hkv": 8, "D": 128, "Tq": 512, "Tk": 4099, "window": 1024, "sinks": 4, "lens": False},
        # A long prompt in one piece.
        {"name": "window_16k", "kind": "window", "B": 1, "Hq": 32, "Hkv": 8, "D": 128, "Tq": 16384, "Tk": 16384, "window": 4096, "sinks": 4, "lens": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "fork", "compact", "decode", "decode", "decode", "window", "window", "window"])
    bits, page, D = rng.choice([4, 8, 16]), rng.choice([16, 32, 64, 128]), rng.choice([64, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    if kind == "append":
        N, pos = _log(rng, 1, 64), rng.randint(0, 300)
        S = rng.choice([1, _log(rng, 1, max(1, 8192 // N))])
        return {"kind": kind, "N": N, "S": S, "Hkv": Hkv, "D": D, "bits": bits, "page": page, "M": (pos + S + page) // page + rng.randint(0, 5), "pos": pos}
    if kind == "fork":
        parents, children, T = rng.randint(1, 8), rng.randint(1, 7), _log(rng, 1, 2500)
        n = -(-T // page)
        return {"kind": kind, "parents": parents, "children": children, "layers": rng.randint(1, 4 if bits == 16 else 8), "T": T, "Hkv": Hkv, "D": D, "bits": bits,
                "page": page, "P": parents * n + parents * children * 2 + rng.randint(0, 40)}
    if kind == "compact":
        rows, T = rng.randint(1, 24), _log(rng, 16, 4096)
        return {"kind": kind, "rows": rows, "layers": rng.randint(1, 2 if bits == 16 else 4), "T": T, "window": _log(rng, 1, 2048), "sinks": rng.choice([0, 1, 4, 17]),
                "Hkv": Hkv, "D": D, "bits": bits, "page": page, "P": rows * -(-T // page) + rng.randint(0, 64)}
    if kind == "decode":
        B = _log(rng, 1, 64)
        T = _log(rng, 1, min(32768, 262144 // B))
        return {"kind": kind, "B": B, "Hq": Hkv * rng.randint(1, 8), "Hkv": Hkv, "D": D, "T": T, "window": rng.choice([0, 0, _log(rng, 1, 4096)]),
                "sinks": rng.choice([0, 1, 4, 100]), "bits": bits, "page": page}
    Tq = _log(rng, 1, 8192)
    Tk = Tq + rng.choice([0, 0, _log(rng, 1, 8192)])
    c = {"kind": kind, "B": rng.choice([1, 1, 2, 3]) if Tk <= 4096 else 1, "Hq": Hkv * rng.randint(1, 4), "Hkv": Hkv, "D": D, "Tq": Tq, "Tk": Tk,
         "window": rng.choice([0, _log(rng, 1, 4096), _log(rng, 1, 4096)]), "sinks": rng.choice([0, 1, 4, 130]), "lens": rng.random() < 0.3}
    while work(c)["flops"] > 9e11:
        c["Tq"] //= 2
    return c


def _lengths(n, T):
    """Ragged lengths that depend on the case alone: T itself first, down to about half of it."""
    return [max(1, T - b * T // (2 * n)) for b in range(n)]


def _visible(length, window, sinks):
    """Cached tokens that the newest token of a sequence sees."""
    return length if window <= 0 or window + sinks >= length else window + sinks


def _pairs(Tq, Tk, window, sinks):
    """(query, key) pairs of a prompt that are visible."""
    return sum(_visible(p + 1, window, sinks) for p in range(max(0, Tk - Tq), Tk))


def _row_bytes(c):
    """Bytes of one token of one head in one pool of the cache."""
    return c["D"] * 2 if c["bits"] == 16 else c["D"] * c["bits"] // 8 + c["D"] // GROUP * 4


def work(c):
    if c["kind"] == "append":
        rows = 2 * c["Hkv"] * sum(_counts(c))
        return {"bytes": rows * (c["D"] * 2 + _row_bytes(c)), "flops": rows * c["D"] * 4}
    page_bytes = 2 * c["layers"] * c["Hkv"] * c["page"] * _row_bytes(c) if "layers" in c else 0
    if c["kind"] == "fork":
        n = c["parents"] * c["children"]
        copied = sum(c["children"] for t in _lengths(c["parents"], c["T"]) if t % c["page"])
        entries = sum(-(-t // c["page"]) for t in _lengths(c["parents"], c["T"])) * c["children"]
        return {"bytes": 2 * copied * page_bytes + entries * 4 * 4 + c["P"] * 4 + n * 40, "flops": 0}
    if c["kind"] == "compact":
        live, pages = 0, 0
        for t in _lengths(c["rows"], c["T"]):
            n = -(-t // c["page"])
            lo, hi = -(-c["sinks"] // c["page"]), max(0, t - c["window"]) // c["page"]
            pages += n
            live += n - max(0, hi - lo)
        # pages of live data behind the first `live` ones, as many as a random placement leaves there
        moved = live * (c["P"] - live) // c["P"]
        return {"bytes": 2 * moved * page_bytes + pages * 8 + c["P"] * 16, "flops": 0}
    if c["kind"] == "decode":
        tok = sum(_visible(t, c["window"], c["sinks"]) for t in _lengths(c["B"], c["T"]))
        return {"bytes": 2 * c["Hkv"] * tok * _row_bytes(c) + c["B"] * c["Hq"] * c["D"] * 4, "flops": 4 * c["D"] * c["Hq"] * tok}
    total = 0
    for t in _prompt_lens(c):
        total += _pairs(c["Tq"], t, c["window"], c["sinks"])
    return {"bytes": c["B"] * c["D"] * 2 * (2 * c["Hq"] * c["Tq"] + 2 * c["Hkv"] * c["Tk"]), "flops": 4 * c["D"] * c["Hq"] * total}


def _counts(c):
    return [max(1, c["S"] - n * c["S"] // (2 * c["N"])) for n in range(c["N"])]


def _prompt_lens(c):
    return _lengths(c["B"], c["Tk"]) if c["lens"] else [c["Tk"]] * c["B"]


# ---------------------------------------------------------------- the packed format

def _pack(x, bits):
    """Affine quantisation of fp32 rows [..., D] in groups of 64: (codes int32, scales bf16, biases bf16), each step rounded to fp32."""
    shape = x.shape
    g = x.reshape(*shape[:-1], shape[-1] // GROUP, GROUP)
    lo, hi = g.amin(-1), g.amax(-1)
    bins = float((1 << bits) - 1)
    neg = lo.abs() > hi.abs()
    scale = torch.clamp((hi - lo) / torch.full_like(lo, bins), min=1e-7)
    scale = torch.where(neg, scale, -scale)
    edge = torch.where(neg, lo, hi)
    q0 = torch.round(edge / scale)
    zero = q0 == 0
    scale = torch.where(zero, scale, edge / torch.where(zero, torch.ones_like(q0), q0))
    bias = torch.where(zero, torch.zeros_like(edge), edge)
    codes = torch.clamp(torch.round((g - bias[..., None]) / scale[..., None]), 0.0, bins).to(I32)
    per = 32 // bits
    codes = codes.reshape(*shape[:-1], shape[-1] // per, per)
    words = codes[..., 0].clone()
    for i in range(1, per):
        words |= codes[..., i] << (i * bits)
    return words, scale.to(BF16), bias.to(BF16)


def _unpack(words, scales, biases, bits, dtype):
    per = 32 // bits
    shift = torch.arange(per, device=words.device, dtype=I32) * bits
    q = ((words[..., None] >> shift) & ((1 << bits) - 1)).to(dtype)
    q = q.reshape(*words.shape[:-1], scales.shape[-1], GROUP)
    v = q * scales.to(dtype)[..., None] + biases.to(dtype)[..., None]
    return v.reshape(*words.shape[:-1], words.shape[-1] * per)


def _pool(g, c, pages):
    """A pool of cache pages with values ~N(0, 1), the rows of a few channels larger, as keys have them."""
    parts = []
    step = max(1, (1 << 26) // (c["Hkv"] * c["page"] * c["D"]))
    for i in range(0, pages, step):
        x = torch.randn((min(step, pages - i), c["Hkv"], c["page"], c["D"]), device="cuda", generator=g)
        x[..., :: c["D"] // 4] *= 3.0
        parts.append((x.to(BF16), None, None) if c["bits"] == 16 else _pack(x.to(BF16).float(), c["bits"]))
    return tuple(None if p[0] is None else torch.cat(p) for p in zip(*parts))


def _tensors(pool):
    return [t for t in pool if t is not None]


def _layers(g, c, st):
    """K and V pools of every layer: views of one allocation for the codes and one each for scales and biases."""
    st["cache"] = [torch.stack(parts) for parts in zip(*[_tensors(_pool(g, c, c["P"])) for _ in range(2 * c["layers"])])]
    st["pools"] = [view for t in st["cache"] for view in t.unbind(0)]


def _table(g, lens, page, M, P):
    """Pages of every sequence at random places of the pool, as a server's pages are after a while."""
    perm = torch.randperm(P, device="cuda", generator=g).to(I32)
    table = torch.full((len(lens), M), -1, dtype=I32, device="cuda")
    refs = torch.zeros(P, dtype=I32, device="cuda")
    at = 0
    for i, t in enumerate(lens):
        n = -(-t // page)
        table[i, :n] = perm[at:at + n]
        at += n
    refs[perm[:at].long()] = 1
    return table, refs


def _ints(values):
    return torch.tensor(values, dtype=I32, device="cuda")


# ---------------------------------------------------------------- inputs

def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(c)
    kind = c["kind"]
    if kind == "window":
        for name, heads, T in (("q", c["Hq"], c["Tq"]), ("k", c["Hkv"], c["Tk"]), ("v", c["Hkv"], c["Tk"])):
            st[name] = torch.randn((c["B"], heads, T, c["D"]), device="cuda", generator=g).to(BF16)
        st["kv_lens"] = _ints(_prompt_lens(c)) if c["lens"] else None
        st["scale"] = c["D"] ** -0.5
        return st
    if kind == "append":
        lens = [c["M"] * c["page"]] * c["N"]
        P = c["N"] * c["M"] + 3
        st["table"], _ = _table(g, lens, c["page"], c["M"], P)
        st["positions"], st["counts"] = torch.full((c["N"],), c["pos"], dtype=I32, device="cuda"), _ints(_counts(c))
        for name in ("dense_k", "dense_v"):
            st[name] = torch.randn((c["N"], c["Hkv"], c["S"], c["D"]), device="cuda", generator=g).to(BF16)
        st["k"], st["v"] = _pool(g, c, P), _pool(g, c, P)
    elif kind == "decode":
        lens = _lengths(c["B"], c["T"])
        M = -(-c["T"] // c["page"]) + 1
        P = sum(-(-t // c["page"]) for t in lens) + 5
        st["table"], _ = _table(g, lens, c["page"], M, P)
        st["lens"] = _ints(lens)
        st["k"], st["v"] = _pool(g, c, P), _pool(g, c, P)
        st["q"] = torch.randn((c["B"], c["Hq"], 1, c["D"]), device="cuda", generator=g).to(BF16)
        st["scale"] = c["D"] ** -0.5
        if own:
            qb = _lib()
            n = qb.kv_pages_decode_attention_workspace_size(c["B"], c["Hq"], c["Hkv"], c["D"])
            st["workspace"] = torch.empty(n, dtype=torch.uint8, device="cuda")
    elif kind == "fork":
        n = c["parents"] * c["children"]
        S = c["parents"] + n
        lens = _lengths(c["parents"], c["T"])
        M = -(-(c["T"] + 1) // c["page"]) + 1
        st["table"], st["refs"] = _table(g, lens + [0] * n, c["page"], M, c["P"])
        st["lens"] = _ints(lens + [0] * n)
        st["src"] = _ints([i // c["children"] for i in range(n)])
        st["dst"] = _ints(list(range(c["parents"], S)))
        st["ones"] = torch.ones(n, dtype=I32, device="cuda")
        _layers(g, c, st)
    else:
        lens = _lengths(c["rows"], c["T"])
        st["table0"], st["refs0"] = _table(g, lens, c["page"], -(-c["T"] // c["page"]) + 1, c["P"])
        st["lens"] = _ints(lens)
        st["rows"] = torch.arange(c["rows"], dtype=I32, device="cuda")
        st["begin"] = torch.full((c["rows"],), c["sinks"], dtype=I32, device="cuda")
        st["end"] = _ints([max(0, t - c["window"]) for t in lens])
        _layers(g, c, st)
    return st


# ---------------------------------------------------------------- plain forms

def _plain_append(s):
    page, S = s["page"], s["S"]
    i = torch.arange(S, device="cuda")
    # tokens behind a sequence's count are not written: its last one takes their place, so that it is written again
    i = torch.minimum(i[None], s["counts"][:, None].long() - 1)
    pos = s["positions"][:, None].long() + i
    pid = torch.gather(s["table"].long(), 1, pos // page).reshape(-1)
    slot = (pos % page).reshape(-1)
    out = []
    for pool, dense in ((s["k"], s["dense_k"]), (s["v"], s["dense_v"])):
        x = torch.gather(dense, 2, i[:, None, :, None].expand(-1, dense.shape[1], -1, dense.shape[3]))
        x = x.transpose(1, 2).reshape(-1, dense.shape[1], dense.shape[3])
        new = (x,) if s["bits"] == 16 else _pack(x.float(), s["bits"])
        for t, v in zip(_tensors(pool), new):
            t[pid, :, slot] = v
            out.append(t)
    return out


def _add_refs(refs, pages, valid, amount):
    refs.index_add_(0, torch.where(valid, pages, torch.zeros_like(pages)).reshape(-1).long(), (valid.to(I32) * amount).reshape(-1))


def _plain_free(table, lens, refs, page, rows, begin=None, end=None):
    rows = rows.long()
    t, n = table[rows], lens[rows]
    b = torch.zeros_like(n) if begin is None else begin
    e = n if end is None else torch.minimum(end, n)
    col = torch.arange(table.shape[1], device="cuda", dtype=I32)[None]
    inside = (col * page >= b[:, None]) & (torch.minimum((col + 1) * page, n[:, None]) <= e[:, None]) & (col * page < n[:, None])
    _add_refs(refs, t, inside & (t >= 0), -1)
    table[rows] = torch.where(inside, torch.full_like(t, -1), t)
    lens[rows] = torch.where(e >= n, torch.minimum(n, b), n)


def _plain_fork(table, lens, refs, page, src, dst):
    src, dst = src.long(), dst.long()
    n = lens[src]
    t = table[src]
    used = (torch.arange(table.shape[1], device="cuda", dtype=I32)[None] * page < n[:, None])
    table[dst] = torch.where(used, t, table[dst])
    lens[dst] = n
    _add_refs(refs, t, used & (t >= 0), 1)
    return n


def _plain_reserve(table, lens, refs, page, rows, counts):
    rows = rows.long()
    n = lens[rows]
    have, want = (n + page - 1) // page, (n + counts + page - 1) // page
    last = torch.gather(table[rows], 1, torch.clamp(have - 1, min=0)[:, None].long())[:, 0]
    shared = (counts > 0) & (n % page != 0) & (refs[torch.clamp(last, min=0).long()] > 1)
    need = want - have + shared.to(I32)
    first = torch.cumsum(need, 0) - need
    free = torch.cumsum((refs == 0).to(I32), 0)
    col = torch.arange(table.shape[1], device="cuda")[None]
    start = (have - shared.to(I32))[:, None]
    fresh = (col >= start) & (col < want[:, None])
    rank = first[:, None] + (col - start)
    pages = torch.searchsorted(free, torch.where(fresh, rank, torch.zeros_like(rank)) + 1).to(I32)
    table[rows] = torch.where(fresh, pages, table[rows])
    copies = torch.stack([last, torch.gather(table[rows], 1, torch.clamp(have - 1, min=0)[:, None].long())[:, 0]], 1)
    copies = torch.where(shared[:, None], copies, torch.full_like(copies, -1))
    _add_refs(refs, last, shared, -1)
    _add_refs(refs, pages, fresh, 1)
    lens[rows] = n + counts
    return n, copies


def _plain_copy(pools, pairs):
    if pairs.shape[0] == 0:
        return
    valid = pairs[:, 0] >= 0
    # pairs that say nothing repeat the first one that does
    stand_in = pairs[torch.argmax(valid.to(I32))].clamp(min=0)
    pairs = torch.where(valid[:, None], pairs, stand_in[None]).long()
    for t in pools:
        t[pairs[:, 1]] = t[pairs[:, 0]]


def _plain_compact(table, refs):
    P = refs.shape[0]
    live = refs > 0
    ids = torch.arange(P, device="cuda")
    n = live.sum()
    tail, hole = live & (ids >= n), ~live & (ids < n)
    rank = torch.cumsum(tail, 0) - 1
    to = torch.searchsorted(torch.cumsum(hole, 0), torch.clamp(rank, min=0) + 1)
    remap = torch.where(tail, to, torch.where(live, ids, torch.full_like(ids, -1)))
    moves = torch.full((P // 2 + 1, 2), -1, dtype=I32, device="cuda")
    at = torch.where(tail, rank, torch.full_like(rank, P // 2))
    moves[at] = torch.where(tail[:, None], torch.stack([ids, remap], 1), torch.full((P, 2), -1, device="cuda")).to(I32)
    new = torch.zeros(P + 1, dtype=I32, device="cuda")
    new[torch.where(live, remap, torch.full_like(ids, P))] = refs * live
    refs.copy_(new[:P])
    table.copy_(torch.where(table >= 0, remap.to(I32)[table.clamp(min=0).long()], torch.full_like(table, -1)))
    return remap.to(I32), moves[: P // 2]


def _masked_softmax(s, keep):
    """Rows that see nothing are zero."""
    s = s.masked_fill(~keep, float("-inf"))
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    e = e.masked_fill(~keep, 0.0)
    return e / torch.clamp(e.sum(-1, keepdim=True), min=1e-30)


def _plain_decode(s):
    B, Hq, _, D = s["q"].shape
    Hkv, page = s["Hkv"], s["page"]
    T = s["table"].shape[1] * page
    pos = torch.arange(T, device="cuda")
    out = torch.empty_like(s["q"])
    for b in range(B):
        pid = s["table"][b].clamp(min=0).long()
        kv = []
        for pool in (s["k"], s["v"]):
            if s["bits"] == 16:
                x = pool[0][pid].float()
            else:
                x = _unpack(pool[0][pid], pool[1][pid], pool[2][pid], s["bits"], torch.float32)
            kv.append(x.transpose(0, 1).reshape(Hkv, T, D))
        n = s["lens"][b]
        keep = pos < n
        if s["window"] > 0:
            keep &= (pos < s["sinks"]) | (pos >= n - s["window"])
        x = torch.matmul(s["q"][b].float().reshape(Hkv, Hq // Hkv, D), kv[0].transpose(1, 2)) * s["scale"]
        out[b] = torch.matmul(_masked_softmax(x, keep), kv[1]).reshape(Hq, 1, D).to(BF16)
    return out


def _plain_window(s):
    B, Hq, Tq, D = s["q"].shape
    Hkv, Tk = s["k"].shape[1], s["k"].shape[2]
    q = s["q"].float().reshape(B, Hkv, Hq // Hkv, Tq, D)
    k, v = s["k"].float()[:, :, None], s["v"].float()[:, :, None]
    lens = torch.full((B,), Tk, device="cuda") if s["kv_lens"] is None else s["kv_lens"].long()
    out = torch.empty_like(s["q"]).reshape(B, Hkv, Hq // Hkv, Tq, D)
    step = 256
    for i in range(0, Tq, step):
        n = min(step, Tq - i)
        hi = Tk if s["kv_lens"] is not None else Tk - Tq + i + n
        at = lens[:, None] - Tq + i + torch.arange(n, device="cuda")[None]
        j = torch.arange(hi, device="cuda")[None, None]
        keep = j <= at[..., None]
        if s["window"] > 0:
            keep &= (j < s["sinks"]) | (j > at[..., None] - s["window"])
        x = torch.matmul(q[..., i:i + n, :], k[..., :hi, :].transpose(-1, -2)) * s["scale"]
        out[..., i:i + n, :] = torch.matmul(_masked_softmax(x, keep[:, None, None]), v[..., :hi, :]).to(BF16)
    return out.reshape(B, Hq, Tq, D)


# ---------------------------------------------------------------- one pass

def run(s):
    kind = s["kind"]
    qb = _lib() if own else None
    if kind == "append":
        if not own:
            return _plain_append(s)
        qb.kv_pages_append(s["k"], s["v"], s["dense_k"], s["dense_v"], s["table"], s["positions"], s["bits"], GROUP, counts=s["counts"])
        return _tensors(s["k"]) + _tensors(s["v"])
    if kind == "decode":
        if not own:
            return _plain_decode(s)
        return qb.kv_pages_decode_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["bits"], GROUP, s["scale"], window=s["window"], sinks=s["sinks"],
                                            workspace=s["workspace"])
    if kind == "window":
        if not own:
            return _plain_window(s)
        return qb.window_attention(s["q"], s["k"], s["v"], s["scale"], window=s["window"], sinks=s["sinks"], kv_lens=s["kv_lens"])
    if kind == "fork":
        table, lens, refs, page = s["table"], s["lens"], s["refs"], s["page"]
        if own:
            qb.kv_pages_free(table, lens, refs, page, s["dst"])
            shared = qb.kv_pages_fork(table, lens, refs, page, s["src"], s["dst"])
            positions, copies = qb.kv_pages_reserve(table, lens, refs, page, s["dst"], s["ones"])
            qb.kv_pages_copy(s["pools"], copies)
        else:
            _plain_free(table, lens, refs, page, s["dst"])
            shared = _plain_fork(table, lens, refs, page, s["src"], s["dst"])
            positions, copies = _plain_reserve(table, lens, refs, page, s["dst"], s["ones"])
            _plain_copy(s["pools"], copies)
        return [table, lens, refs, shared, positions, copies] + s["cache"]
    # the state before the pass comes back first: a compact pool has nothing to compact
    table, refs, lens, page = s["table0"].clone(), s["refs0"].clone(), s["lens"].clone(), s["page"]
    if own:
        qb.kv_pages_free(table, lens, refs, page, s["rows"], s["begin"], s["end"])
        remap, moves, count = qb.kv_pages_compact(table, refs)
        qb.kv_pages_copy(s["pools"], moves, count)
    else:
        _plain_free(table, lens, refs, page, s["rows"], s["begin"], s["end"])
        remap, moves = _plain_compact(table, refs)
        _plain_copy(s["pools"], moves)
    return [table, refs, lens, remap, moves] + s["cache"]


# ---------------------------------------------------------------- in 64 bits

def exact(c, seed):
    """From the definition: every output row as one sum over the tokens that it sees.  Page bookkeeping and packed rows are
    whole numbers, which have no other value in 64 bits."""
    if c["kind"] not in ("decode", "window"):
        return None
    s = prepare(c, seed)
    F64 = torch.float64
    rep = c["Hq"] // c["Hkv"]
    if c["kind"] == "decode":
        out = torch.zeros(s["q"].shape, dtype=F64, device="cuda")
        for b, n in enumerate(_lengths(c["B"], c["T"])):
            seen = [t for t in range(n) if c["window"] <= 0 or t < c["sinks"] or t >= n - c["window"]]
            at = torch.tensor(seen, device="cuda")
            page, slot = s["table"][b][at // c["page"]].long(), at % c["page"]
            rows = []
            for pool in (s["k"], s["v"]):
                part = [t[page, :, slot] for t in _tensors(pool)]
                rows.append(part[0].to(F64) if c["bits"] == 16 else _unpack(*part, c["bits"], F64))
            for h in range(c["Hkv"]):
                x = s["q"][b, h * rep:(h + 1) * rep, 0].to(F64) @ rows[0][:, h].T * s["scale"]
                out[b, h * rep:(h + 1) * rep, 0] = torch.softmax(x, -1) @ rows[1][:, h]
        return out
    out = torch.zeros(s["q"].shape, dtype=F64, device="cuda")
    for b, n in enumerate(_prompt_lens(c)):
        for i in range(0, c["Tq"], 1024):
            at = torch.arange(n - c["Tq"] + i, n - c["Tq"] + min(i + 1024, c["Tq"]), device="cuda")[:, None]
            j = torch.arange(n, device="cuda")[None]
            hidden = j > at
            if c["window"] > 0:
                hidden |= (j >= c["sinks"]) & (j <= at - c["window"])
            for h in range(c["Hq"]):
                x = s["q"][b, h, i:i + 1024].to(F64) @ s["k"][b, h // rep, :n].to(F64).T * s["scale"]
                p = torch.softmax(x.masked_fill(hidden, -math.inf), -1).masked_fill(hidden, 0.0)
                out[b, h, i:i + 1024] = p @ s["v"][b, h // rep, :n].to(F64)
    return out
