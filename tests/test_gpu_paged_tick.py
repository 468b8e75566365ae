"""The paged cache as a server uses it: prompts through the projections and the prompt attention into pages, forked answers, and ticks of
projections, reserve, copy, append, attention and output projection -- called one by one, and as a captured graph that is replayed."""
import pytest
import torch

import qb200

pytestmark = pytest.mark.gpu
I32, BF16 = torch.int32, torch.bfloat16
HID, HQ, HKV, D, PAGE, M, P, SEQS, WINDOW, SINKS = 512, 8, 2, 64, 16, 12, 60, 5, 40, 4


def ints(*x):
    return torch.tensor(x, dtype=I32, device="cuda")


class Server:
    def __init__(self, bits, layers=2):
        g = torch.Generator(device="cuda").manual_seed(3)
        rnd = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF16)
        self.bits = bits
        self.w = [[qb200.quantize(rnd(n, HID) * 0.05, 64, 4) for n in (HQ * D, HKV * D, HKV * D, HID)] for _ in range(layers)]
        self.table = torch.full((SEQS, M), -1, dtype=I32, device="cuda")
        self.lens, self.refs = torch.zeros(SEQS, dtype=I32, device="cuda"), torch.zeros(P, dtype=I32, device="cuda")

        def pool():
            if bits == 16:
                return (torch.zeros(P, HKV, PAGE, D, dtype=BF16, device="cuda"), None, None)
            return (torch.zeros(P, HKV, PAGE, D * bits // 32, dtype=I32, device="cuda"), *(torch.zeros(P, HKV, PAGE, D // 64, dtype=BF16, device="cuda") for _ in range(2)))

        self.kv = [(pool(), pool()) for _ in range(layers)]
        self.pools = [t for pair in self.kv for side in pair for t in side if t is not None]
        self.ws = torch.empty(qb200.kv_pages_decode_attention_workspace_size(SEQS, HQ, HKV, D), dtype=torch.uint8, device="cuda")

    def project(self, x, w):
        return qb200.quantized_matmul(x, *w, group_size=64, bits=4)

    def heads(self, y, n):
        return y.view(y.shape[0], y.shape[1], n, D).transpose(1, 2)

    def prompt(self, row, x):
        """x [1, T, HID] into sequence `row`."""
        T = x.shape[1]
        pos, copies = qb200.kv_pages_reserve(self.table, self.lens, self.refs, PAGE, ints(row), ints(T))
        qb200.kv_pages_copy(self.pools, copies)
        for (wq, wk, wv, wo), (kp, vp) in zip(self.w, self.kv):
            q, k, v = self.heads(self.project(x, wq), HQ), self.heads(self.project(x, wk), HKV), self.heads(self.project(x, wv), HKV)
            o = qb200.window_attention(q, k, v, D ** -0.5, window=WINDOW, sinks=SINKS)
            qb200.kv_pages_append(kp, vp, k, v, self.table, pos, self.bits, rows=ints(row))
            x = self.project(o.transpose(1, 2).reshape(1, T, HQ * D), wo)
        return x

    def tick(self, x, rows, ones):
        """x [n, 1, HID]: a token of each listed sequence."""
        pos, copies = qb200.kv_pages_reserve(self.table, self.lens, self.refs, PAGE, rows, ones)
        qb200.kv_pages_copy(self.pools, copies)
        for (wq, wk, wv, wo), (kp, vp) in zip(self.w, self.kv):
            q, k, v = self.heads(self.project(x, wq), HQ), self.heads(self.project(x, wk), HKV), self.heads(self.project(x, wv), HKV)
            qb200.kv_pages_append(kp, vp, k, v, self.table, pos, self.bits, rows=rows)
            o = qb200.kv_pages_decode_attention(q, kp, vp, self.table, self.lens, self.bits, 64, D ** -0.5, window=WINDOW, sinks=SINKS, rows=rows, workspace=self.ws)
            x = self.project(o.transpose(1, 2).reshape(x.shape[0], 1, HQ * D), wo)
        return x

    def state(self):
        return [self.table, self.lens, self.refs] + self.pools


def start(bits):
    s = Server(bits)
    g = torch.Generator(device="cuda").manual_seed(5)
    first = [s.prompt(r, torch.randn(1, T, HID, device="cuda", generator=g).to(BF16)) for r, T in ((0, 77), (3, 130))]
    assert qb200.kv_pages_fork(s.table, s.lens, s.refs, PAGE, ints(0, 0), ints(1, 2)).tolist() == [77, 77]
    return s, first


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_a_captured_tick_gives_what_the_calls_give(bits):
    (one, _), (two, _) = start(bits), start(bits)
    rows, ones = ints(2, 0, 3, 1), ints(1, 1, 1, 1)
    x = torch.empty(4, 1, HID, dtype=BF16, device="cuda")
    spare, _ = start(bits)                       # (first calls set their kernels up; they are made on another state)
    spare.tick(torch.zeros_like(x), rows, ones)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            y = two.tick(x, rows, ones)
            x.copy_(y / y.float().abs().amax(-1, keepdim=True).clamp(min=1e-6).to(BF16))
    token = torch.randn(4, 1, HID, device="cuda", generator=torch.Generator(device="cuda").manual_seed(8)).to(BF16)
    x.copy_(token)
    torch.cuda.synchronize()
    for step in range(20):                       # (past the ends of pages, and of the window)
        want = one.tick(token, rows, ones)
        token = want / want.float().abs().amax(-1, keepdim=True).clamp(min=1e-6).to(BF16)
        with torch.cuda.stream(s):
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.view(torch.int16), want.view(torch.int16)), step
        for a, b in zip(one.state(), two.state()):
            assert torch.equal(a, b), step
    assert one.lens.tolist() == [97, 97, 97, 150, 0] and bool(torch.isfinite(want).all())
    assert qb200.lib().qb200_debug_tc_status() == 0


def test_forked_answers_of_equal_tokens_stay_equal_and_others_part():
    s, _ = start(8)
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(1, 1, HID, device="cuda", generator=g).to(BF16).expand(3, 1, HID).contiguous()
    y = s.tick(x, ints(0, 1, 2), ints(1, 1, 1))
    assert torch.equal(y[0], y[1]) and torch.equal(y[0], y[2])
    x[2] += 1
    y = s.tick(x, ints(0, 1, 2), ints(1, 1, 1))
    assert torch.equal(y[0], y[1]) and not torch.equal(y[0], y[2])
    # the pages that left the window go; what the window sees stays, and so do the results
    twin, _ = start(8)
    for t in (x * 0 + 1, x):
        twin.tick(t, ints(0, 1, 2), ints(1, 1, 1))
    s2, _ = start(8)
    for t in (x * 0 + 1, x):
        s2.tick(t, ints(0, 1, 2), ints(1, 1, 1))
    end = (s2.lens[:3] - WINDOW).contiguous()
    before = int((s2.refs > 0).sum())
    qb200.kv_pages_free(s2.table, s2.lens, s2.refs, PAGE, ints(0, 1, 2), begin=ints(SINKS, SINKS, SINKS), end=end)
    remap, moves, count = qb200.kv_pages_compact(s2.table, s2.refs)
    qb200.kv_pages_copy(s2.pools, moves, count)
    assert int((s2.refs > 0).sum()) < before
    for t in (x, x + 2):
        assert torch.equal(s2.tick(t, ints(1, 0, 2), ints(1, 1, 1)), twin.tick(t, ints(1, 0, 2), ints(1, 1, 1)))
