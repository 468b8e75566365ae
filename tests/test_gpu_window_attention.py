"""GPU tests of the prompt attention with a window and sinks, against fp64.

Tolerance of one output o = sum p v: half a bf16 step of the result; the probabilities rounded to bf16 (half a step, 2^-8) and the
exponential's error (at most 2^-13 of each, in the sum too), against A = sum p |v|; the scores' fp32 sums of D products, 2^-20 of
S = scale * sum |q| |k| as the exponent's absolute error, against A too."""
import pytest
import torch

import qb200

pytestmark = pytest.mark.gpu
I32, BF16, F64 = torch.int32, torch.bfloat16, torch.float64


def visible(Tq, n, window, sinks):
    p = (n - Tq + torch.arange(Tq, device="cuda"))[:, None]
    j = torch.arange(n, device="cuda")[None]
    see = j <= p
    if window > 0:
        see &= (j > p - window) | (j < sinks)
    return see


def check(out, q, k, v, scale, window=0, sinks=0, lens=None, poisoned=None):
    B, Hq, Tq, D = q.shape
    rep = Hq // k.shape[1]
    for b in range(B):
        n = k.shape[2] if lens is None else max(0, min(lens[b], k.shape[2]))
        see = visible(Tq, n, window, sinks)
        none = ~see.any(1)
        for h in range(Hq):
            qh, kh, vh, got = q[b, h].to(F64), k[b, h // rep, :n].to(F64), v[b, h // rep, :n].to(F64), out[b, h].to(F64)
            s = (qh @ kh.T * scale).masked_fill(~see, float("-inf"))
            p = torch.softmax(s, -1).masked_fill(~see, 0.0)
            o, A = p @ vh, p @ vh.abs()
            S = (qh.abs() @ kh.abs().T * scale).masked_fill(~see, 0.0).amax(-1, keepdim=True) if n else torch.zeros(Tq, 1, device="cuda", dtype=F64)
            tol = 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2 * 2.0 ** -13 + 2.0 ** -20 * S) * A + 1e-30
            o[none], tol[none] = 0.0, 0.0
            ok = torch.ones(Tq, dtype=torch.bool, device="cuda") if poisoned is None else ~poisoned(b, h // rep, see)
            assert not torch.isnan(got[ok]).any(), f"b {b} h {h}: NaN"
            worst = ((got - o).abs()[ok] / (tol[ok] + 1e-30)).max().item() if ok.any() else 0.0
            assert worst <= 1.01, f"b {b} h {h}: {worst:.2f} of the tolerance"
            if poisoned is not None:
                assert torch.isnan(got[~ok]).all()


def make(B, Hq, Hkv, Tq, Tk, D, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(B, h, T, D, device="cuda", generator=g) * std).to(BF16) for h, T in ((Hq, Tq), (Hkv, Tk), (Hkv, Tk))]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Hq,Hkv,Tq,Tk", [(1, 2, 1, 1, 1), (1, 2, 2, 77, 77), (2, 4, 2, 128, 128), (1, 3, 1, 129, 300), (1, 2, 1, 300, 300), (1, 1, 1, 513, 700), (3, 6, 2, 5, 400), (1, 2, 1, 1, 1000)])
def test_causal(D, B, Hq, Hkv, Tq, Tk):
    q, k, v = make(B, Hq, Hkv, Tq, Tk, D)
    check(qb200.window_attention(q, k, v, D ** -0.5), q, k, v, D ** -0.5)


@pytest.mark.parametrize("D,gqa", [(64, 2), (128, 1), (128, 4)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (17, 0), (128, 4), (129, 128), (200, 130), (300, 500), (699, 1), (10 ** 12, 2), (64, 10 ** 12), (0, 5)])
@pytest.mark.parametrize("Tq,Tk", [(700, 700), (200, 831)])
def test_window_and_sinks(D, gqa, window, sinks, Tq, Tk):
    q, k, v = make(1, 2 * gqa, 2, Tq, Tk, D, window % 101)
    check(qb200.window_attention(q, k, v, D ** -0.5, window=window, sinks=sinks), q, k, v, D ** -0.5, window, sinks)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Hq,Hkv,Tq,Tk,window,sinks", [(1, 2, 1, 1, 5000, 0, 0), (1, 4, 4, 130, 3000, 0, 0), (1, 8, 2, 300, 4099, 1024, 4), (3, 2, 1, 100, 2000, 700, 200)])
@pytest.mark.parametrize("clusters", [True, False])
def test_tiles_whose_keys_several_blocks_share(D, B, Hq, Hkv, Tq, Tk, window, sinks, clusters, request):
    if not clusters:
        request.getfixturevalue("no_clusters")
    q, k, v = make(B, Hq, Hkv, Tq, Tk, D, Tq)
    lens = None if B == 1 else [2000, 55, 0]
    out = qb200.window_attention(q, k, v, D ** -0.5, window=window, sinks=sinks, kv_lens=None if lens is None else torch.tensor(lens, dtype=I32, device="cuda"))
    check(out, q, k, v, D ** -0.5, window, sinks, lens)
    assert qb200.lib().qb200_debug_tc_status() == 0


def test_a_long_prompt():
    q, k, v = make(1, 4, 2, 3000, 5000, 128)
    for window, sinks in ((0, 0), (1024, 4)):
        check(qb200.window_attention(q, k, v, 128 ** -0.5, window=window, sinks=sinks), q, k, v, 128 ** -0.5, window, sinks)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 5)])
def test_lengths_from_the_device(D, window, sinks):
    """Queries before position 0 give zeros; keys and values behind a length, NaN here, are not seen."""
    lens = [400, 250, 130, 1, 0, 1000, -3]
    q, k, v = make(7, 2, 1, 200, 400, D)
    for b, n in enumerate(lens):
        k[b, :, max(n, 0):], v[b, :, max(n, 0):] = float("nan"), float("nan")
    out = qb200.window_attention(q, k, v, 0.1, window=window, sinks=sinks, kv_lens=torch.tensor(lens, dtype=I32, device="cuda"))
    check(out, q, k, v, 0.1, window, sinks, lens)


@pytest.mark.parametrize("D,gqa", [(64, 1), (128, 2)])
def test_what_is_not_finite_shows_where_it_is_seen_and_nowhere_else(D, gqa):
    Tq, Tk, window, sinks = 400, 600, 100, 3
    q, k, v = make(1, 2 * gqa, 2, Tq, Tk, D)
    bad = {0: [(150, float("nan")), (599, float("inf")), (340, float("-inf"))], 1: [(1, float("nan")), (260, float("inf"))]}
    for h, rows in bad.items():
        for j, x in rows:
            v[0, h, j, 7] = x
    v[0, :, 50], k[0, :, 60] = float("nan"), float("nan")           # no query sees these
    out = qb200.window_attention(q, k, v, 0.1, window=window, sinks=sinks)
    clean = torch.nan_to_num(v, 0.0, 0.0, 0.0)
    poisoned = lambda b, h, see: see[:, [j for j, _ in bad[h]]].any(1)
    # (in blocks that a query sees whole the value itself comes through, so only that it is not finite is asked of all channels together)
    fine = torch.where(torch.isfinite(out).all(-1, keepdim=True), out, torch.full_like(out, float("nan")))
    check(fine, q, torch.nan_to_num(k), clean, 0.1, window, sinks, poisoned=poisoned)
    assert qb200.lib().qb200_debug_tc_status() == 0
    k2 = torch.nan_to_num(k)
    k2[0, 1, 333, 3] = float("nan")
    out = qb200.window_attention(q, k2, clean, 0.1, window=window, sinks=sinks)
    check(out, q, torch.nan_to_num(k), clean, 0.1, window, sinks, poisoned=lambda b, h, see: see[:, 333] if h == 1 else torch.zeros(Tq, dtype=torch.bool, device="cuda"))


@pytest.mark.parametrize("std", [1e-3, 8.0])
def test_magnitudes(std):
    """Flat softmax rows, and rows whose maximum grows by far more than the reference may lie behind."""
    q, k, v = make(1, 2, 1, 500, 500, 128, 3, std)
    k *= torch.linspace(0, 2, 500, device="cuda").to(BF16)[None, None, :, None]
    check(qb200.window_attention(q, k, v, 0.1), q, k, v, 0.1)


def test_strides_and_broadcast():
    D = 64
    qkv = torch.randn(2, 300, 8, D + 8, device="cuda").to(BF16)            # [B, T, heads, .] as a projection leaves it
    q, k, v = (qkv[:, :, a:b, :D].transpose(1, 2) for a, b in ((0, 4), (4, 6), (6, 8)))
    res = torch.full((2, 4, 300, D + 3), 9.0, device="cuda", dtype=BF16)
    qb200.window_attention(q, k, v, 0.2, window=70, sinks=2, out=res[..., 1:D + 1])
    check(res[..., 1:D + 1], q, k, v, 0.2, 70, 2)
    assert bool((res[..., 0] == 9).all()) and bool((res[..., D + 1:] == 9).all())
    one_k, one_v = k[:1, :1].expand(2, 2, 300, D), v[:1, :1].expand(2, 2, 300, D)     # one head for all, one sequence for all
    check(qb200.window_attention(q, one_k, one_v, 0.2), q, one_k, one_v, 0.2)
    check(qb200.window_attention(q[:1].expand(2, 4, 300, D), k, v, 0.2), q[:1].expand(2, 4, 300, D), k, v, 0.2)


def test_rows_of_other_sequences_do_not_leak():
    """Keys of the next head or sequence follow in memory: a length that ends inside a block of 128."""
    q, k, v = make(2, 2, 2, 130, 130, 128)
    k[1], v[1], k[:, 1], v[:, 1] = 50.0, 1e4, 50.0, 1e4
    k[0, 0], v[0, 0] = torch.randn(130, 128, device="cuda").to(BF16), torch.randn(130, 128, device="cuda").to(BF16)
    out = qb200.window_attention(q, k, v, 0.1)
    check(out[:1, :1], q[:1, :1], k[:1, :1], v[:1, :1], 0.1)


def test_the_last_query_agrees_with_the_paged_call():
    """A prompt's last position and one new token over pages of the same rows."""
    H, D, T, page = 2, 128, 777, 64
    q, k, v = make(1, 8, H, T, T, D)
    out = qb200.window_attention(q, k, v, D ** -0.5, window=300, sinks=4)
    M = -(-T // page)
    pool = []
    for x in (k, v):
        p = torch.zeros(M, H, page, D, device="cuda", dtype=BF16)
        table = torch.arange(M, device="cuda", dtype=I32)[None]
        pool.append((p, None, None))
    qb200.kv_pages_append(*pool, k, v, table, torch.zeros(1, dtype=I32, device="cuda"), 16)
    one = qb200.kv_pages_decode_attention(q[:, :, -1:], *pool, table, torch.tensor([T], dtype=I32, device="cuda"), 16, 64, D ** -0.5, window=300, sinks=4)
    check(one, q[:, :, -1:], k, v, D ** -0.5, 300, 4)
    check(out[:, :, -1:], q[:, :, -1:], k, v, D ** -0.5, 300, 4)


def test_streams_graphs_and_the_status_word():
    q, k, v = make(1, 4, 2, 700, 700, 128)
    lens = torch.tensor([700], dtype=I32, device="cuda")
    out = torch.empty_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            qb200.window_attention(q, k, v, 0.1, window=300, sinks=4, kv_lens=lens, out=out)
    for n in (700, 333, 0):
        lens.fill_(n)
        torch.cuda.synchronize()
        g.replay()
        again = qb200.window_attention(q, k, v, 0.1, window=300, sinks=4, kv_lens=lens)
        torch.cuda.synchronize()
        check(out, q, k, v, 0.1, 300, 4, [n])
        assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    assert qb200.lib().qb200_debug_tc_status() == 0


def test_sequences_far_apart():
    """Sequences and heads whose elements lie beyond 2^31 of each other, in every operand and in the result."""
    D, far = 64, 2 ** 31 + 64
    q, k, v = make(2, 2, 2, 140, 140, D)
    res = torch.zeros_like(q)

    def spread(x, axis):
        x = x.contiguous()
        stride = [far if i == axis else s for i, s in enumerate(x.stride())]
        flat = torch.empty(far + x.stride(0) * 2, dtype=BF16, device="cuda")
        y = flat.as_strided(x.shape, stride)
        y.copy_(x)
        return y

    for axis in (0, 1):
        fq, fk, fv, fr = (spread(x, axis) for x in (q, k, v, res))
        qb200.window_attention(fq, fk, fv, 0.1, window=50, sinks=3, out=fr)
        check(fr, q, k, v, 0.1, 50, 3)


def crowd(q, k, v, *args, lens=None, **kw):
    """The call on so many copies of its sequences that every CTA takes two tiles; all copies give the same."""
    n = 160 // (q.shape[0] * q.shape[1]) + 1
    rep = lambda x: x.repeat(n, 1, 1, 1)
    if lens is not None:
        kw["kv_lens"] = torch.tensor(lens * n, dtype=I32, device="cuda")
    out = qb200.window_attention(rep(q), rep(k), rep(v), *args, **kw).view(n, *q.shape)
    bits = out.view(torch.int16)
    assert torch.equal(bits, bits[:1].expand_as(bits))
    return out[0]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(2, 1), (3, 1), (2, 2)])
@pytest.mark.parametrize("Tq,Tk,window,sinks", [(1, 1, 0, 0), (77, 77, 32, 2), (129, 300, 0, 0), (256, 256, 1, 0), (300, 700, 200, 130), (513, 513, 129, 128), (140, 900, 64, 10 ** 12)])
def test_two_tiles_a_block(D, Hq, Hkv, Tq, Tk, window, sinks):
    q, k, v = make(1, Hq, Hkv, Tq, Tk, D, Tq)
    check(crowd(q, k, v, D ** -0.5, window=window, sinks=sinks), q, k, v, D ** -0.5, window, sinks)


@pytest.mark.parametrize("D,gqa,window,sinks", [(64, 1, 0, 0), (128, 2, 90, 5), (128, 3, 90, 5)])
def test_two_tiles_a_block_with_lengths(D, gqa, window, sinks):
    lens = [400, 250, 130, 1, 0, 1000, -3]
    q, k, v = make(7, gqa, 1, 200, 400, D)
    for b, n in enumerate(lens):
        k[b, :, max(n, 0):], v[b, :, max(n, 0):] = float("nan"), float("nan")
    check(crowd(q, k, v, 0.1, window=window, sinks=sinks, lens=lens), q, k, v, 0.1, window, sinks, lens)


@pytest.mark.parametrize("D,gqa", [(64, 1), (128, 2)])
def test_two_tiles_a_block_and_what_is_not_finite(D, gqa):
    Tq, Tk, window, sinks = 400, 600, 100, 3
    q, k, v = make(1, 2 * gqa, 2, Tq, Tk, D)
    bad = {0: [(150, float("nan")), (599, float("inf")), (340, float("-inf"))], 1: [(1, float("nan")), (260, float("inf"))]}
    for h, rows in bad.items():
        for j, x in rows:
            v[0, h, j, 7] = x
    v[0, :, 50], k[0, :, 60] = float("nan"), float("nan")           # no query sees these
    out = crowd(q, k, v, 0.1, window=window, sinks=sinks)
    clean = torch.nan_to_num(v, 0.0, 0.0, 0.0)
    poisoned = lambda b, h, see: see[:, [j for j, _ in bad[h]]].any(1)
    fine = torch.where(torch.isfinite(out).all(-1, keepdim=True), out, torch.full_like(out, float("nan")))
    check(fine, q, torch.nan_to_num(k), clean, 0.1, window, sinks, poisoned=poisoned)


@pytest.mark.parametrize("std", [1e-3, 8.0])
def test_two_tiles_a_block_of_any_magnitude(std):
    q, k, v = make(1, 2, 1, 500, 500, 128, 3, std)
    k *= torch.linspace(0, 2, 500, device="cuda").to(BF16)[None, None, :, None]
    check(crowd(q, k, v, 0.1), q, k, v, 0.1)


def test_a_long_prompt_of_many_heads():
    q, k, v = make(1, 16, 2, 3000, 5000, 128)
    for window, sinks in ((0, 0), (1024, 4)):
        check(qb200.window_attention(q, k, v, 128 ** -0.5, window=window, sinks=sinks), q, k, v, 128 ** -0.5, window, sinks)
    assert qb200.lib().qb200_debug_tc_status() == 0


@pytest.mark.parametrize("B,Hq,Hkv,Tq,Tk,D,window,sinks,lens", [
    (1, 32, 8, 256, 4096, 128, 0, 0, None), (1, 28, 4, 250, 4099, 64, 0, 0, None), (1, 32, 8, 500, 16384, 128, 0, 0, None),
    (4, 8, 4, 200, 4096, 128, 0, 0, [4096, 3001, 150, 0]), (1, 32, 8, 200, 6000, 128, 4000, 300, None)])
@pytest.mark.parametrize("clusters", [True, False])
def test_two_tiles_a_block_whose_keys_several_blocks_share(B, Hq, Hkv, Tq, Tk, D, window, sinks, lens, clusters, request):
    """More tiles than fit one a block with as many clusters; a value that is not finite shows in the heads that see it."""
    if not clusters:
        request.getfixturevalue("no_clusters")
    q, k, v = make(B, Hq, Hkv, Tq, Tk, D, Tq)
    kl = None if lens is None else torch.tensor(lens, dtype=I32, device="cuda")
    call = lambda v: qb200.window_attention(q, k, v, D ** -0.5, window=window, sinks=sinks, kv_lens=kl)
    out = call(v)
    check(out, q, k, v, D ** -0.5, window, sinks, lens)
    bad = v.clone()
    n = Tk if lens is None else lens[0]
    bad[0, 1, n - 1, 5] = float("inf")                        # seen by the last query alone
    bits = call(bad).view(torch.int16) != out.view(torch.int16)
    g = Hq // Hkv
    assert bool(bits[0, g:2 * g, -1].any(-1).all())
    bits[0, g:2 * g, -1] = False
    assert not bool(bits.any())
    assert qb200.lib().qb200_debug_tc_status() == 0
