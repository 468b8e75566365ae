"""A round of decoding with drafted tokens over the paged key-value cache, as cases that can be timed: attention of a tree of drafted
tokens over pages, sampling a token from each row of logits, and the walk that keeps the drafted tokens which the samples confirm.

A case is a dict of plain values; ``kind`` picks the operator.  With ``own`` false ``run`` computes in elementary torch operations in
fp32 (sums of probabilities, which are compared with one another, in 64 bits); with ``own`` true it makes the library's calls.  Head
layouts and lengths are those of this repository's benchmark configurations (32 query heads on 8 cache heads of 128, caches of 32k
tokens, 16 sequences) and of its tests (7 query heads to a cache head, head dim 64, odd lengths); page sizes, windows, trees and
vocabularies are generic.

Cache pages: a pool is [pages, heads, page, cols]; at 4 and 8 bits a triple of packed codes (int32 words, lowest bits first),
bf16 scales and biases per 64 values, at 16 bits the bf16 rows themselves.  ``table`` [sequences, pages of a sequence] holds page
numbers, -1 where there is none; ``lens`` the tokens of a sequence, the drafted ones among them: the last ``counts`` tokens are the
nodes of the tree, ``parents`` says behind which node each stands (-1: behind the cached tokens), always one before it.
"""
import math
import os
import random
import sys

import torch

own = False
BF16, I32, F32, F64 = torch.bfloat16, torch.int32, torch.float32, torch.float64
GROUP = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _lib():
    path = os.path.abspath("mlx-serve_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import qb200
    return qb200


# ---------------------------------------------------------------- cases

def listed():
    return [
        # One user, a short context, four tokens drafted in a chain: the smallest call, where the fixed part counts.
        {"name": "tree_1_chain", "kind": "tree", "B": 1, "Hq": 32, "Hkv": 8, "D": 128, "T": 700, "nodes": 4, "chain": True, "window": 0, "sinks": 0, "bits": 4, "page": 64},
        # Thirteen users of different lengths with up to 16 drafted tokens each, seven query heads to a cache head, 8 bits, small pages.
        {"name": "tree_13_ragged", "kind": "tree", "B": 13, "Hq": 28, "Hkv": 4, "D": 128, "T": 8191, "nodes": 16, "chain": False, "window": 0, "sinks": 0, "bits": 8,
         "page": 16},
        # A layer with a window over an unquantised cache: 32 users, eight drafted tokens each.
        {"name": "tree_32_window", "kind": "tree", "B": 32, "Hq": 64, "Hkv": 8, "D": 64, "T": 16384, "nodes": 8, "chain": False, "window": 1024, "sinks": 4, "bits": 16,
         "page": 128},
        # Three users, odd sizes all through: 27 nodes, 5 query heads to a cache head, bf16 rows.
        {"name": "tree_3_odd", "kind": "tree", "B": 3, "Hq": 15, "Hkv": 3, "D": 128, "T": 2049, "nodes": 27, "chain": False, "window": 0, "sinks": 0, "bits": 16, "page": 32},
        # Four users with the widest trees, 64 nodes, over 8k tokens at 8 bits.
        {"name": "tree_4_wide", "kind": "tree", "B": 4, "Hq": 32, "Hkv": 8, "D": 128, "T": 8192, "nodes": 64, "chain": False, "window": 0, "sinks": 0, "bits": 8, "page": 64},
        # Sixteen users of up to 32k tokens at 4 bits, 32 nodes each: the largest read of the cache.
        {"name": "tree_16_32k", "kind": "tree", "B": 16, "Hq": 32, "Hkv": 8, "D": 128, "T": 32768, "nodes": 32, "chain": False, "window": 0, "sinks": 0, "bits": 4, "page": 64},
        # One user's next token with the usual filters: latency.
        {"name": "sample_1", "kind": "sample", "N": 1, "V": 128256, "dtype": "bf16", "temperature": 0.7, "top_k": 50, "top_p": 0.95, "min_p": 0.0, "masked": False,
         "logprobs": True},
        # The nodes of sixteen trees, every row with settings of its own (greedy ones among them), a part of the vocabulary masked.
        {"name": "sample_256_mixed", "kind": "sample", "N": 256, "V": 32001, "dtype": "fp32", "temperature": "mixed", "top_k": "mixed", "top_p": "mixed", "min_p": "mixed",
         "masked": True, "logprobs": True},
        # A nucleus over a flat distribution: tens of thousands of tokens are kept.
        {"name": "sample_24_nucleus", "kind": "sample", "N": 24, "V": 151667, "dtype": "fp16", "temperature": 1.5, "top_k": 0, "top_p": 0.95, "min_p": 0.0, "masked": False,
         "logprobs": True},
        # A large batch over a large vocabulary by temperature alone: the logits are what there is to read.
        {"name": "sample_256_plain", "kind": "sample", "N": 256, "V": 262144, "dtype": "bf16", "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "masked": False,
         "logprobs": False},
        # Four users' walks through trees of eight, rows of two layers moved: latency.
        {"name": "accept_4", "kind": "accept", "B": 4, "nodes": 8, "layers": 2, "T": 700, "Hkv": 8, "D": 128, "bits": 4, "page": 64},
        # Sixteen users' walks through trees of 48, the rows of sixteen layers moved.
        {"name": "accept_16", "kind": "accept", "B": 16, "nodes": 48, "layers": 16, "T": 1000, "Hkv": 8, "D": 128, "bits": 8, "page": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "tree", "sample", "sample", "sample", "accept"])
    bits, page, D, Hkv = rng.choice([4, 8, 16]), rng.choice([16, 32, 64, 128]), rng.choice([64, 128]), rng.choice([1, 2, 4, 8])
    if kind == "tree":
        B = _log(rng, 1, 32)
        c = {"kind": kind, "B": B, "Hq": Hkv * rng.randint(1, 8), "Hkv": Hkv, "D": D, "T": _log(rng, 1, min(32768, 262144 // B)), "nodes": _log(rng, 1, 64),
             "chain": rng.random() < 0.3, "window": rng.choice([0, 0, _log(rng, 1, 4096)]), "sinks": rng.choice([0, 1, 4, 100]), "bits": bits, "page": page}
        while work(c)["flops"] > 2e11:
            c["T"] //= 2
        return c
    if kind == "sample":
        V = _log(rng, 2, 262144)
        return {"kind": kind, "N": min(_log(rng, 1, 512), (1 << 25) // V), "V": V, "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "temperature": rng.choice(["mixed", 0.0, round(rng.uniform(0.2, 2.0), 2)]), "top_k": rng.choice(["mixed", 0, _log(rng, 1, 2000)]),
                "top_p": rng.choice(["mixed", 1.0, round(rng.uniform(0.05, 1.0), 3)]), "min_p": rng.choice(["mixed", 0.0, round(rng.uniform(0.0, 0.3), 3)]),
                "masked": rng.random() < 0.3, "logprobs": rng.random() < 0.5}
    return {"kind": kind, "B": _log(rng, 1, 64), "nodes": _log(rng, 1, 64), "layers": rng.randint(1, 8), "T": _log(rng, 1, 2000), "Hkv": Hkv, "D": D, "bits": bits,
            "page": page}


def _lengths(c):
    """Ragged lengths that depend on the case alone, the nodes among them: the longest first, down to about half of it."""
    return [max(n, c["T"] - b * c["T"] // (2 * c["B"])) for b, n in enumerate(_counts(c))]


def _counts(c):
    return [max(1, c["nodes"] - b * c["nodes"] // (2 * c["B"])) for b in range(c["B"])]


def _parents(c, seed):
    """The trees: parents before their nodes; half of the nodes stand behind one of the last few, so that the trees are deep as well as wide."""
    rng = random.Random(seed)
    trees = []
    for n in _counts(c):
        t = [-1]
        while len(t) < n:
            t.append(len(t) - 1 if c.get("chain") else rng.randrange(max(0, len(t) - 4), len(t)) if rng.random() < 0.5 else rng.randrange(len(t)))
        trees.append(t)
    return trees


def _visible(length, window, sinks):
    """Tokens that the last token of a sequence sees."""
    return length if window <= 0 or window + sinks >= length else window + sinks


def _row_bytes(c):
    """Bytes of one token of one head in one pool of the cache."""
    return c["D"] * 2 if c["bits"] == 16 else c["D"] * c["bits"] // 8 + c["D"] // GROUP * 4


def work(c):
    if c["kind"] == "tree":
        keys = pairs = rows = 0
        for n, t in zip(_counts(c), _lengths(c)):
            keys += _visible(t, c["window"], c["sinks"])
            # a node sees the cached tokens and, in a tree like these, about a dozen of its ancestors
            pairs += n * _visible(t - n + min(n, 12), c["window"], c["sinks"])
            rows += n
        return {"bytes": 2 * c["Hkv"] * keys * _row_bytes(c) + rows * c["Hq"] * c["D"] * 4, "flops": 4 * c["D"] * c["Hq"] * pairs}
    if c["kind"] == "sample":
        return {"bytes": c["N"] * (c["V"] * (4 if c["dtype"] == "fp32" else 2) + 24), "flops": 10 * c["N"] * c["V"]}
    # about half of a path's tokens stand elsewhere than where they go
    moved = sum(min(n, 6) // 2 for n in _counts(c))
    return {"bytes": 2 * moved * 2 * c["layers"] * c["Hkv"] * _row_bytes(c) + c["B"] * c["nodes"] * 4 * 5, "flops": 0}


# ---------------------------------------------------------------- the packed format

def _pack(x, bits):
    """Codes of bf16 rows [..., D] in groups of 64, by the group's smallest and largest value: (codes int32, scales bf16, biases bf16)."""
    g = x.float().reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = g.amin(-1), g.amax(-1)
    scale = ((hi - lo) / (2 ** bits - 1)).clamp(min=1e-7).to(BF16)
    bias = lo.to(BF16)
    codes = torch.round((g - bias.float()[..., None]) / scale.float()[..., None]).clamp(0, 2 ** bits - 1).to(I32)
    per = 32 // bits
    codes = codes.reshape(*x.shape[:-1], -1, per)
    words = codes[..., 0].clone()
    for i in range(1, per):
        words |= codes[..., i] << (i * bits)
    return words, scale, bias


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
        parts.append((x.to(BF16), None, None) if c["bits"] == 16 else _pack(x.to(BF16), c["bits"]))
    return tuple(None if p[0] is None else torch.cat(p) for p in zip(*parts))


def _tensors(pool):
    return [t for t in pool if t is not None]


def _table(g, lens, page, M, P):
    """Pages of every sequence at random places of the pool, as a server's pages are after a while."""
    perm = torch.randperm(P, device="cuda", generator=g).to(I32)
    table = torch.full((len(lens), M), -1, dtype=I32, device="cuda")
    at = 0
    for i, t in enumerate(lens):
        n = -(-t // page)
        table[i, :n] = perm[at:at + n]
        at += n
    return table


def _ints(values):
    return torch.tensor(values, dtype=I32, device="cuda")


def _padded(lists, width, fill=-1):
    return _ints([x + [fill] * (width - len(x)) for x in lists])


# ---------------------------------------------------------------- inputs

MIXED = {"temperature": [0.0, 0.7, 1.0, 1.3, 0.3], "top_k": [40, 0, 1, 500], "top_p": [0.9, 1.0, 0.5], "min_p": [0.0, 0.05]}


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(c)
    if c["kind"] == "sample":
        N, V = c["N"], c["V"]
        # most of the vocabulary around zero, a few tokens of every row well above it, as a trained model's logits lie
        x = torch.empty((N, V), device="cuda", dtype=DTYPES[c["dtype"]])
        for i in range(0, N, 64):
            part = torch.randn((min(64, N - i), V), device="cuda", generator=g) * 2.5
            few = torch.randint(0, V, (part.shape[0], min(V, 12)), device="cuda", generator=g)
            part.scatter_add_(1, few, torch.rand(few.shape, device="cuda", generator=g) * 12.0)
            if c["masked"]:
                out = torch.rand(part.shape, device="cuda", generator=g) < 0.4
                part.masked_fill_(out, torch.finfo(x.dtype).min if i % 128 else -math.inf)
            x[i:i + 64] = part.clamp(torch.finfo(x.dtype).min, None) if c["masked"] and i % 128 else part
        st["logits"] = x
        st["random"] = torch.rand(N, device="cuda", generator=g)
        for name, kinds in MIXED.items():
            value = c[name]
            values = [kinds[i % len(kinds)] for i in range(N)] if value == "mixed" else [value] * N
            st[name] = torch.tensor(values, dtype=I32 if name == "top_k" else F32, device="cuda")
        return st
    lens, page = _lengths(c), c["page"]
    P = sum(-(-t // page) for t in lens) + 5
    st["table"] = _table(g, lens, page, -(-max(lens) // page) + 1, P)
    st["lens"], st["counts"] = _ints(lens), _ints(_counts(c))
    trees = _parents(c, seed)
    st["parents"] = _padded(trees, c["nodes"])
    if c["kind"] == "tree":
        st["k"], st["v"] = _pool(g, c, P), _pool(g, c, P)
        st["q"] = torch.randn((c["B"], c["Hq"], c["nodes"], c["D"]), device="cuda", generator=g).to(BF16)
        st["scale"] = c["D"] ** -0.5
        if own:
            qb = _lib()
            n = qb.kv_pages_tree_attention_workspace_size(c["B"], c["Hq"], c["Hkv"], c["nodes"], c["D"])
            st["workspace"] = torch.empty(n, dtype=torch.uint8, device="cuda")
        return st
    # Drafted tokens, and what was sampled behind each node: along one path down the tree the next node's token, so that a few are kept.
    rng = random.Random(seed + 1)
    tokens, sampled = [], []
    for t in trees:
        ids = [rng.randrange(32000) for _ in t]
        behind = [rng.randrange(32000) for _ in t]
        at = 0
        for _ in range(rng.randrange(1, 8)):
            children = [i for i, p in enumerate(t) if p == at]
            if not children:
                break
            child = rng.choice(children)
            behind[at] = ids[child]
            at = child
        tokens.append(ids)
        sampled.append(behind)
    st["tokens"], st["sampled"] = _padded(tokens, c["nodes"]), _padded(sampled, c["nodes"])
    st["cache"] = [torch.stack(parts) for parts in zip(*[_tensors(_pool(g, c, P)) for _ in range(2 * c["layers"])])]
    st["pools"] = [view for t in st["cache"] for view in t.unbind(0)]
    return st


# ---------------------------------------------------------------- plain forms

def _ancestors(parents):
    """sees[b, t, a]: node a is node t or stands before it; depths of the nodes."""
    B, T = parents.shape
    sees = torch.eye(T, dtype=torch.bool, device="cuda").expand(B, T, T).clone()
    up = parents.long()
    for _ in range(T):
        ok = up >= 0
        sees.scatter_(2, torch.where(ok, up, torch.arange(T, device="cuda"))[..., None], True)
        up = torch.where(ok, torch.gather(parents.long(), 1, up.clamp(min=0)), up)
    return sees, sees.sum(-1) - 1


def _masked_softmax(s, keep):
    """Rows that see nothing are zero."""
    s = s.masked_fill(~keep, float("-inf"))
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    e = e.masked_fill(~keep, 0.0)
    return e / torch.clamp(e.sum(-1, keepdim=True), min=1e-30)


def _plain_tree(s):
    B, Hq, N, D = s["q"].shape
    Hkv, page = s["Hkv"], s["page"]
    T = s["table"].shape[1] * page
    pos = torch.arange(T, device="cuda")
    sees, depth = _ancestors(s["parents"])
    out = torch.empty_like(s["q"])
    for b in range(B):
        pid = s["table"][b].clamp(min=0).long()
        kv = []
        for pool in (s["k"], s["v"]):
            x = pool[0][pid].float() if s["bits"] == 16 else _unpack(pool[0][pid], pool[1][pid], pool[2][pid], s["bits"], F32)
            kv.append(x.transpose(0, 1).reshape(Hkv, T, D))
        base = s["lens"][b] - s["counts"][b]
        node = pos - base
        drafted = (node >= 0) & (node < s["counts"][b])
        at = torch.where(drafted, base + depth[b][node.clamp(0, N - 1)], pos)
        mine = base + depth[b]
        keep = torch.where(drafted[None], sees[b][:, node.clamp(0, N - 1)], (pos < base)[None])
        if s["window"] > 0:
            keep = keep & ((at < s["sinks"])[None] | (at[None] > mine[:, None] - s["window"]))
        keep = keep & (torch.arange(N, device="cuda") < s["counts"][b])[:, None]
        x = torch.matmul(s["q"][b].float().reshape(Hkv, Hq // Hkv * N, D), kv[0].transpose(1, 2)) * s["scale"]
        p = _masked_softmax(x.reshape(Hkv, Hq // Hkv, N, T), keep)
        out[b] = torch.matmul(p.reshape(Hkv, -1, T), kv[1]).reshape(Hq, N, D).to(BF16)
    return out


def _plain_sample(s):
    x = s["logits"].float()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    N, V = x.shape
    value, index = torch.sort(x, dim=1, descending=True, stable=True)
    first = index[:, 0]
    t = s["temperature"].double()[:, None]
    sampling = t > 0
    top = value[:, :1]
    w = torch.exp((value.double() - top.double().clamp(min=-1e300)) / torch.where(sampling, t, torch.ones_like(t)))
    # (a row of which everything is masked has nothing to choose from: -1)
    w = torch.where(value == top, torch.ones_like(w), w) * (value > -math.inf)
    rank = torch.arange(V, device="cuda")[None]
    k = s["top_k"].long()[:, None]
    w = torch.where((k <= 0) | (rank < k), w, torch.zeros_like(w))
    before = torch.cumsum(w, 1) - w
    p = s["top_p"].double()[:, None]
    w = torch.where((p >= 1) | (before < p * w.sum(1, keepdim=True)) | (rank == 0), w, torch.zeros_like(w))
    w = torch.where((w >= s["min_p"].double()[:, None]) | (rank == 0), w, torch.zeros_like(w))
    w = torch.zeros_like(w).scatter_(1, index, w)
    upto = torch.cumsum(w, 1)
    at = torch.searchsorted(upto, s["random"].double()[:, None] * upto[:, -1:], right=True)[:, 0]
    token = torch.where(sampling[:, 0], at.clamp(max=V - 1), first)
    some = top[:, 0] > -math.inf
    tokens = torch.where(some, token, torch.full_like(token, -1)).to(I32)
    if not s["logprobs"]:
        return tokens
    # of the chosen token, before temperature and filters
    d = torch.where(x == top, torch.zeros_like(x), x - top.clamp(min=-3e38))
    chosen = torch.gather(d, 1, token[:, None])[:, 0]
    return [tokens, torch.where(some, chosen - torch.log(torch.exp(d).sum(1, dtype=F64)).float(), torch.zeros_like(chosen))]


def _plain_accept(s):
    B, T = s["parents"].shape
    rows = torch.arange(B, device="cuda")
    parents, tokens, sampled = s["parents"].long(), s["tokens"], s["sampled"]
    live = torch.arange(T, device="cuda")[None] < s["counts"][:, None]
    path = torch.full((B, T), -1, dtype=torch.long, device="cuda")
    path[:, 0] = 0
    at = torch.zeros(B, dtype=torch.long, device="cuda")
    going = torch.ones(B, dtype=torch.bool, device="cuda")
    for i in range(1, T):
        child = (parents == at[:, None]) & (tokens == sampled[rows, at][:, None]) & live
        going = going & child.any(1)
        at = torch.where(going, torch.argmax(child.to(I32), 1), at)
        path[:, i] = torch.where(going, at, path[:, i])
    accepted = (path >= 0).sum(1)
    base = (s["lens"] - s["counts"]).long()
    new = torch.where(path >= 0, torch.gather(sampled, 1, path.clamp(min=0)), torch.full_like(sampled, -1))
    page = s["page"]
    # a place behind the path keeps its row
    src = base[:, None] + torch.where(path >= 0, path, torch.arange(T, device="cuda")[None])
    dst = base[:, None] + torch.arange(T, device="cuda")[None]
    inside = live.reshape(-1)
    where = []
    for pos in (src, dst):
        pos = torch.where(live, pos, base[:, None])
        where += [torch.gather(s["table"].long(), 1, pos // page).reshape(-1), (pos % page).reshape(-1)]
    # entries behind a sequence's nodes take the place of its first
    first = torch.div(torch.arange(B * T, device="cuda"), T, rounding_mode="floor") * T
    pick = torch.where(inside, torch.arange(B * T, device="cuda"), first)
    where = [w[pick] for w in where]
    for t in s["pools"]:
        t[where[2], :, where[3]] = t[where[0], :, where[1]]
    return [path.to(I32), new.to(I32), accepted.to(I32), (base + accepted).to(I32)]


# ---------------------------------------------------------------- one pass

def run(s):
    kind = s["kind"]
    qb = _lib() if own else None
    if kind == "tree":
        if not own:
            return _plain_tree(s)
        return qb.kv_pages_tree_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["parents"], s["bits"], GROUP, s["scale"], window=s["window"],
                                          sinks=s["sinks"], counts=s["counts"], workspace=s["workspace"])
    if kind == "sample":
        if not own:
            return _plain_sample(s)
        return qb.sample(s["logits"], s["random"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], want_logprobs=s["logprobs"])
    if own:
        out = list(qb.kv_pages_accept(s["pools"], s["table"], s["lens"], s["page"], s["parents"], s["tokens"], s["sampled"], counts=s["counts"]))
    else:
        out = _plain_accept(s)
    return out + s["cache"]


# ---------------------------------------------------------------- in 64 bits

def exact(c, seed):
    """From the definitions.  Attention: every output row as one sum over the tokens that it sees.  Sampling: the kept tokens one filter
    after the other by comparing with a border value.  The walk and the rows that it moves have no other value in 64 bits."""
    if c["kind"] == "accept":
        return None
    s = prepare(c, seed)
    if c["kind"] == "sample":
        out, logprobs = [], []
        for i in range(c["N"]):
            x = s["logits"][i].to(F64)
            if i:
                logprobs.append(float(last[out[-1]] - torch.logsumexp(last, 0)) if out[-1] >= 0 else 0.0)
            last = x
            t, k, p, least = (s[n][i].item() for n in ("temperature", "top_k", "top_p", "min_p"))
            ids = torch.nonzero(x > -math.inf)[:, 0]
            order = ids[torch.argsort(-x[ids], stable=True)]
            if t <= 0 or len(order) == 0:
                out.append(int(order[0]) if len(order) else -1)
                continue
            if k > 0:
                order = order[:k]
            w = torch.exp((x[order] - x[order[0]]) / t)
            if p < 1:
                share = torch.cumsum(w, 0)
                order = order[:max(1, int((share < p * share[-1]).sum()) + 1)]
                w = w[:len(order)]
            stay = w >= least
            stay[0] = True
            order, w = order[stay], w[stay]
            by_index = torch.argsort(order)
            upto = torch.cumsum(w[by_index], 0)
            at = min(int((upto <= s["random"][i].item() * upto[-1]).sum()), len(order) - 1)
            out.append(int(order[by_index[at]]))
        logprobs.append(float(last[out[-1]] - torch.logsumexp(last, 0)) if out[-1] >= 0 else 0.0)
        return [_ints(out), torch.tensor(logprobs, dtype=F64, device="cuda")] if c["logprobs"] else _ints(out)
    rep = c["Hq"] // c["Hkv"]
    out = torch.zeros(s["q"].shape, dtype=F64, device="cuda")
    for b, (n, length, tree) in enumerate(zip(_counts(c), _lengths(c), _parents(c, seed))):
        base = length - n
        depth, line = [], []
        for t, p in enumerate(tree):
            depth.append(0 if p < 0 else depth[p] + 1)
            line.append([t] if p < 0 else line[p] + [t])
        where = torch.arange(length, device="cuda")
        page, slot = s["table"][b][where // c["page"]].long(), where % c["page"]
        rows = []
        for pool in (s["k"], s["v"]):
            part = [x[page, :, slot] for x in _tensors(pool)]
            rows.append(part[0].to(F64) if c["bits"] == 16 else _unpack(*part, c["bits"], F64))
        for t in range(n):
            me = base + depth[t]
            inside = lambda at: c["window"] <= 0 or at < c["sinks"] or at > me - c["window"]
            if c["window"] <= 0:
                old = torch.arange(base, device="cuda")
            else:
                start = max(0, me - c["window"] + 1)
                old = torch.cat([torch.arange(min(c["sinks"], start, base), device="cuda"), torch.arange(min(start, base), base, device="cuda")])
            drafted = [base + a for a in line[t] if inside(base + depth[a])]
            seen = torch.cat([old, torch.tensor(drafted, dtype=torch.long, device="cuda")])
            for h in range(c["Hkv"]):
                x = s["q"][b, h * rep:(h + 1) * rep, t].to(F64) @ rows[0][seen, h].T * s["scale"]
                out[b, h * rep:(h + 1) * rep, t] = torch.softmax(x, -1) @ rows[1][seen, h]
    return out
