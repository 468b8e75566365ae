"""GPU tests of the attention of one new token over pages, against fp64 on the values that the codes stand for.

Tolerance of one output o = sum p v, from the kernel's roundings: half a bf16 step of the result; the probabilities times the scaled
codes rounded to fp16 (half a step, 2^-11) or to two bf16 (2^-16), against A = sum p |code part|; the scores' fp32 sums, about ten
roundings of 2^-24 of S = scale * sum |q| |k| + the approximate exponential's 2^-22 twice, against B = sum p (|code part| + |bias|)."""
import numpy as np
import pytest
import torch

import qb200
from pages_ref import F64, decode, seen

pytestmark = pytest.mark.gpu
I32, BF16 = torch.int32, torch.bfloat16


def ints(x):
    return torch.tensor(x, dtype=I32, device="cuda")


def unpack(pool, bits):
    """(code part, bias part) of every row, fp64 [P, H, page, D]."""
    if bits == 16:
        v = pool[0].to(F64)
        return v, torch.zeros_like(v)
    w, s, b = pool
    q = ((w[..., None].to(torch.int64) >> (torch.arange(32 // bits, device="cuda") * bits)) & (2 ** bits - 1)).reshape(*w.shape[:-1], -1)
    rep = lambda x: x.to(F64).repeat_interleave(64, -1)
    return q.to(F64) * rep(s), rep(b).expand(q.shape)


def make_pool(P, H, page, D, bits, std=1.0):
    x = (torch.randn(P, H, page, D, device="cuda") * std).to(BF16)
    return (x, None, None) if bits == 16 else qb200.quantize(x, 64, bits)


def make_table(lens, page, M, P, seed=0):
    perm = np.random.default_rng(seed).permutation(P).tolist()
    return [[perm.pop() if p * page < n else -1 for p in range(M)] for n in lens]


def check(out, q, kp, vp, table, lens, page, bits, scale, window=0, sinks=0, rows=None, no_page=lambda e: e < 0):
    B, Hq, _, D = q.shape
    (kc, kb), (vc, vb) = unpack(kp, bits), unpack(vp, bits)
    H = kc.shape[1]
    half = 2.0 ** -16 if bits == 16 else 2.0 ** -11
    got = out.to(F64).cpu().numpy()
    qs = q.to(F64).cpu().numpy()
    for b in range(B):
        r = b if rows is None else rows[b]
        n = max(0, min(lens[r], len(table[r]) * page)) if 0 <= r < len(table) else 0
        keep = [t for t in seen(n, window, sinks) if not no_page(table[r][t // page])]
        at = torch.tensor(keep, device="cuda", dtype=torch.long)
        pid = torch.tensor([table[r][t // page] for t in keep], device="cuda", dtype=torch.long)
        g = [x[pid, :, at % page].cpu().numpy() for x in (kc, kb, vc, vb)]
        for h in range(Hq):
            hk = h // (Hq // H)
            k, v, a = g[0][:, hk] + g[1][:, hk], g[2][:, hk] + g[3][:, hk], np.abs(g[2][:, hk])
            o, p = decode(qs[b, h, 0], k, v, scale, np.arange(len(keep)))
            assert not np.isnan(got[b, h, 0]).any()
            if not keep:
                assert (got[b, h, 0] == 0).all()
                continue
            S = float((abs(scale) * (np.abs(g[0][:, hk]) + np.abs(g[1][:, hk])) @ np.abs(qs[b, h, 0])).max())
            tol = 2.0 ** -8 * np.abs(o) + half * (p @ a) + (10 * 2.0 ** -24 * S + 2.0 ** -21) * (p @ (a + np.abs(g[3][:, hk]))) + 1e-30
            err = np.abs(got[b, h, 0] - o)
            assert (err <= tol * 1.01).all(), f"b {b} h {h}: worst {float((err / tol).max()):.2f} of the tolerance"


def run(kp, vp, table, lens, bits, B, Hq, D, seed=0, **kw):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(B, Hq, 1, D, device="cuda", generator=g).to(BF16)
    return q, qb200.kv_pages_decode_attention(q, kp, vp, ints(table), ints(lens), bits, 64, D ** -0.5, **kw)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("D,H,gqa,page,lens", [
    (128, 2, 4, 64, [1, 63, 64, 65, 200]), (64, 1, 1, 16, [17, 0, 130]), (128, 4, 7, 32, [300, 5]), (64, 8, 8, 128, [129, 128]), (128, 1, 11, 16, [77]), (64, 2, 16, 256, [700, 1])])
def test_lengths_heads_and_pages(bits, D, H, gqa, page, lens):
    torch.manual_seed(bits)
    M = max(-(-n // page) for n in lens) + 1
    P = sum(-(-n // page) for n in lens) + 3
    kp, vp = make_pool(P, H, page, D, bits), make_pool(P, H, page, D, bits)
    table = make_table(lens, page, M, P)
    q, out = run(kp, vp, table, lens, bits, len(lens), H * gqa, D)
    check(out, q, kp, vp, table, lens, page, bits, D ** -0.5)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (33, 4), (64, 64), (100, 130), (500, 0), (200, 3), (10 ** 12, 4), (0, 9), (70, 10 ** 12)])
def test_window_and_sinks(bits, window, sinks):
    torch.manual_seed(window % 97 + sinks % 89)
    lens, page, D, H = [400, 333, 64, 3, 0], 32, 128, 2
    M, P = 14, 40
    kp, vp = make_pool(P, H, page, D, bits), make_pool(P, H, page, D, bits)
    table = make_table(lens, page, M, P)
    q, out = run(kp, vp, table, lens, bits, 5, 8, D, window=window, sinks=sinks)
    check(out, q, kp, vp, table, lens, page, bits, D ** -0.5, window, sinks)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("B,T,page,H,gqa,D,window,sinks", [(1, 9000, 64, 2, 4, 128, 0, 0), (3, 5000, 16, 8, 3, 64, 0, 0), (40, 700, 32, 2, 8, 128, 0, 0), (7, 6000, 128, 4, 5, 128, 2000, 70),
                                                           (200, 90, 16, 1, 2, 64, 0, 0)])
def test_sequences_that_several_blocks_share(bits, B, T, page, H, gqa, D, window, sinks):
    torch.manual_seed(T)
    lens = [max(0, T - (i * T * 5) // (4 * B)) for i in range(B)]
    M, P = -(-T // page), sum(-(-n // page) for n in lens) + 1
    kp, vp = make_pool(P, H, page, D, bits), make_pool(P, H, page, D, bits)
    table = make_table(lens, page, M, P)
    q, out = run(kp, vp, table, lens, bits, B, H * gqa, D, window=window, sinks=sinks)
    check(out, q, kp, vp, table, lens, page, bits, D ** -0.5, window, sinks)


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_rows_strides_and_lengths_outside_the_table(bits):
    """Queries of listed sequences (one twice, one that does not exist), lengths above the capacity and below zero, pools with the heads
    inside the page, queries and results with strides, scale rows off 16 bytes."""
    torch.manual_seed(5)
    S, page, M, P, H, D = 4, 16, 5, 30, 2, 64
    lens, rows = [70, 1000, -4, 33], [3, 1, 1, 7, 2, -1, 0]
    kp, vp = make_pool(P, H, page, D, bits), make_pool(P, H, page, D, bits)
    table = make_table([80, 80, 80, 33], page, M, P)
    heads = lambda p: tuple(None if t is None else t.transpose(1, 2).contiguous().transpose(1, 2) for t in p)
    off = lambda p: p if bits == 16 else (p[0], *(torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape) for t in p[1:]))
    wide = torch.randn(7, 6, 2, D + 5, device="cuda").to(BF16)
    q = wide[:, :, 1:, 3:3 + D]
    res = torch.full((7, 12, 1, D), 9.0, device="cuda", dtype=BF16)
    for k, v in ((kp, vp), (heads(kp), heads(vp)), (off(kp), vp), (kp, off(heads(vp)))):
        out = res[:, ::2]
        qb200.kv_pages_decode_attention(q, k, v, ints(table), ints(lens), bits, 64, 0.2, rows=ints(rows), out=out)
        check(out, q, kp, vp, table, lens, page, bits, 0.2, rows=rows)
        assert bool((res[:, 1::2] == 9.0).all())


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_what_is_not_seen_is_not_read(bits):
    """NaN and infinities in pages and rows that no query sees: behind the length, between sinks and window, in pages that the table
    does not name; entries that are no page are not seen."""
    torch.manual_seed(6)
    page, M, P, H, D, n, window, sinks = 32, 12, 20, 2, 128, 333, 90, 5
    kp, vp = make_pool(P, H, page, D, bits), make_pool(P, H, page, D, bits)
    table = make_table([M * page], page, M, P)
    bad = [t for t in range(M * page) if t not in set(seen(n, window, sinks))]
    for i, t in enumerate(bad):
        for pool in (kp, vp):
            for x in (pool[:1] if bits == 16 else pool[1:]):
                x[table[0][t // page], :, t % page] = [float("nan"), float("inf"), float("-inf")][i % 3]
    table[0][9], table[0][2], table[0][10] = -1, P, -5      # (page 10 holds the newest rows)
    clean = [tuple(None if t is None else torch.nan_to_num(t, 0.0, 0.0, 0.0) if t.dtype == BF16 else t for t in p) for p in (kp, vp)]
    for pages in (set(), {8}):
        tab = [[e if i not in pages else -1 for i, e in enumerate(table[0])]]
        q, out = run(kp, vp, tab, [n], bits, 1, 8, D, window=window, sinks=sinks)
        check(out, q, *clean, tab, [n], page, bits, D ** -0.5, window, sinks, no_page=lambda e: not 0 <= e < P)
    q, out = run(kp, vp, [[-1] * M], [n], bits, 1, 8, D)
    assert bool((out == 0).all())


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_what_is_seen_and_not_finite_shows(bits):
    torch.manual_seed(7)
    kp, vp = make_pool(8, 2, 16, 64, bits), make_pool(8, 2, 16, 64, bits)
    (kp[0] if bits == 16 else kp[1])[3, 1, 5] = float("nan")
    q, out = run(kp, vp, [[3, 1], [2, 0]], [20, 20], bits, 2, 4, 64)
    assert bool(torch.isnan(out[0, 2:]).all()) and not bool(torch.isnan(out[0, :2]).any()) and not bool(torch.isnan(out[1]).any())
    kp, vp = make_pool(8, 2, 16, 64, bits), make_pool(8, 2, 16, 64, bits)
    q[1, 3, 0, 7] = float("inf")
    out = qb200.kv_pages_decode_attention(q, kp, vp, ints([[3, 1], [2, 0]]), ints([20, 20]), bits, 64, 0.1)
    assert bool(torch.isnan(out[1, 3]).all()) and not bool(torch.isnan(out[1, :3]).any()) and not bool(torch.isnan(out[0]).any())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("kstd,vstd,qstd", [(1e-3, 1e-6, 1.0), (30.0, 1e4, 1.0), (1.0, 1.0, 1e-20), (1e-2, 1e5, 1e3)])
def test_magnitudes(bits, kstd, vstd, qstd):
    """Values far from 1 on every side: the power-of-two scalings keep to fp16's range."""
    torch.manual_seed(8)
    page, D, H, lens = 32, 128, 2, [500, 90]
    kp, vp = make_pool(40, H, page, D, bits, kstd), make_pool(40, H, page, D, bits, vstd)
    vp[1][3:9] *= 1e-4
    vp[2][3:9] *= 1e-4
    table = make_table(lens, page, 16, 40)
    q = (torch.randn(2, 8, 1, D, device="cuda") * qstd).to(BF16)
    out = qb200.kv_pages_decode_attention(q, kp, vp, ints(table), ints(lens), bits, 64, D ** -0.5)
    check(out, q, kp, vp, table, lens, page, bits, D ** -0.5)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30])
def test_scales_of_either_sign(bits, scale):
    torch.manual_seed(11)
    page, D, H, lens = 32, 64, 2, [300, 90]
    kp, vp = make_pool(40, H, page, D, bits), make_pool(40, H, page, D, bits)
    table = make_table(lens, page, 16, 40)
    q = torch.randn(2, 8, 1, D, device="cuda").to(BF16)
    out = qb200.kv_pages_decode_attention(q, kp, vp, ints(table), ints(lens), bits, 64, scale, window=100, sinks=5)
    check(out, q, kp, vp, table, lens, page, bits, scale, 100, 5)


def test_constant_values_without_scale():
    """Value scales of zero over a long context: the softmax's sum stays finite."""
    D, page, n = 64, 64, 5000
    P = -(-n // page)
    kp, vp = make_pool(P, 1, page, D, 4, 1e-3), make_pool(P, 1, page, D, 4)
    vp[1].zero_()
    vp[2].fill_(0.75)
    q, out = run(kp, vp, [list(range(P))], [n], 4, 1, 2, D)
    assert bool((out == 0.75).all())


def test_the_paged_call_agrees_with_the_contiguous_one():
    """The same codes in capacity buffers and in pages."""
    torch.manual_seed(9)
    B, H, D, T, page = 3, 4, 128, 900, 64
    lens = [900, 311, 64]
    k, v = (qb200.quantize(torch.randn(B, H, 960, D, device="cuda").to(BF16), 64, 4) for _ in range(2))
    q = torch.randn(B, 16, 1, D, device="cuda").to(BF16)
    want = qb200.kv_decode_attention(q, k, v, 4, 64, 0.09, kv_lens=ints(lens))
    to_pages = lambda t: t.reshape(B, H, 15, page, -1).transpose(1, 2).reshape(B * 15, H, page, -1).contiguous()
    out = qb200.kv_pages_decode_attention(q, [to_pages(t) for t in k], [to_pages(t) for t in v], ints([[15 * b + i for i in range(15)] for b in range(B)]), ints(lens), 4, 64, 0.09)
    # each is within half a bf16 step and 2^-11 of the values' size of the exact one
    assert float((out.float() - want.float()).abs().max()) <= float(want.float().abs().max()) * 2.0 ** -7 + 2 * 2.0 ** -11 * 4


def test_replayed_graphs_streams_and_repeated_calls():
    """A captured call replayed after the lengths, the table and the rows changed; two streams with a workspace each; the same bits
    every time."""
    torch.manual_seed(10)
    B, H, D, page, M, bits = 4, 2, 128, 16, 40, 4
    P = B * M
    kp, vp = make_pool(P, H, page, D, bits), make_pool(P, H, page, D, bits)
    table, lens = ints(make_table([M * page] * B, page, M, P)), ints([640, 100, 7, 500])
    q = torch.randn(B, 8, 1, D, device="cuda").to(BF16)
    n = qb200.kv_pages_decode_attention_workspace_size(B, 8, H, D)
    ws = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for _ in range(2)]
    out = torch.empty_like(q)
    call = lambda o, w: qb200.kv_pages_decode_attention(q, kp, vp, table, lens, bits, 64, 0.1, workspace=w, out=o)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call(out, ws[0])
            call(out, ws[0])
    for new in ([640, 100, 7, 500], [1, 0, 640, 333]):
        lens.copy_(ints(new))
        table.copy_(table.flip(0))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check(out, q, kp, vp, table.tolist(), new, page, bits, 0.1)
        again, other = torch.empty_like(q), torch.empty_like(q)
        torch.cuda.synchronize()
        for _ in range(5):
            call(again, ws[0])
            with torch.cuda.stream(s):
                call(other, ws[1])
        torch.cuda.synchronize()
        assert torch.equal(again.view(torch.int16), out.view(torch.int16)) and torch.equal(other.view(torch.int16), out.view(torch.int16))


@pytest.mark.parametrize("bits", [4, 16])
def test_pages_far_apart(bits):
    """Pages half a gigabyte apart: written, copied and read at offsets beyond 32 bits, of elements and of bytes."""
    torch.manual_seed(8)
    P, H, page, D, lens = 20, 2, 32, 128, [200, 77, 64]

    def far(shape, dtype):
        stride = 2 ** 29 // dtype.itemsize
        inner = shape[1] * shape[2] * shape[3]
        flat = torch.empty((P - 1) * stride + inner, dtype=dtype, device="cuda")
        return flat.as_strided(shape, [stride, shape[2] * shape[3], shape[3], 1])

    def pool():
        if bits == 16:
            p = (far([P, H, page, D], BF16), None, None)
        else:
            p = (far([P, H, page, D * bits // 32], I32), far([P, H, page, D // 64], BF16), far([P, H, page, D // 64], BF16))
        for x in p:
            if x is not None:
                x.zero_()
        return p

    kp, vp = pool(), pool()
    table = [[19, 0, 17, 3, 18, 9, 15], [12, 14, 16] + [-1] * 4, [13, 11] + [-1] * 5]
    dense = [torch.randn(3, H, 200, D, device="cuda").to(BF16) for _ in range(2)]
    qb200.kv_pages_append(kp, vp, *dense, ints(table), ints([0, 0, 0]), bits, counts=ints(lens))
    qb200.kv_pages_copy([x for x in (*kp, *vp) if x is not None], ints([[19, 1], [0, 10], [16, 8]]))
    table[0][0], table[0][1], table[1][2] = 1, 10, 8
    q, out = run(kp, vp, table, lens, bits, 3, 8, D)
    check(out, q, kp, vp, table, lens, page, bits, D ** -0.5)
    for x, pl in zip(dense, (kp, vp)):                       # the rows, bit for bit as qb200.quantize makes them
        for want, got in zip((x,) if bits == 16 else qb200.quantize(x, 64, bits), pl):
            for b, n in enumerate(lens):
                rows = torch.stack([got[table[b][t // page], :, t % page] for t in range(n)], 1)
                assert torch.equal(rows, want[b, :, :n])


def test_more_sequences_than_the_smaller_forms_hold():
    """The cut of the work over 600 and 1024 sequences, empty ones among them, lengths in shared memory."""
    torch.manual_seed(9)
    for B in (600, 1024):
        lens = [(i * 37) % 90 for i in range(B)]
        page, H, D = 16, 1, 64
        M, P = 6, sum(-(-n // 16) for n in lens)
        kp, vp = make_pool(P, H, page, D, 8), make_pool(P, H, page, D, 8)
        table = make_table(lens, page, M, P)
        q, out = run(kp, vp, table, lens, 8, B, 2, D)
        check(out, q, kp, vp, table, lens, page, 8, D ** -0.5)
