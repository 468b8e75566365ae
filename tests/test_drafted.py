"""What the entries on drafted tokens and the sampling refuse, without a GPU: through the C ABI with descriptors, and by the Python binding."""
import ctypes as C

import pytest
import torch

import qb200 as q
from drafted_ref import line_of, sample, visible, walk
from test_kv_pages import BF16, I32, NONE, pool, ref, t

F32, F16 = q.FLOAT32, q.FLOAT16


def attend(res=None, qq=None, k=None, v=None, table=None, rows=NONE, lens=None, parents=None, counts=NONE, bits=4, gs=64, scale=0.1, window=0, sinks=0, ws=0x1000,
           n=1 << 30):
    k, v = k or pool(), v or pool()
    qq = qq or t(BF16, [3, 4, 5, 128])
    return q.lib().qb200_kv_pages_tree_attention(*ref(res or qq, qq, *k, *v, table or t(I32, [3, 4]), rows, lens or t(I32, [3]), parents or t(I32, [3, 5]), counts),
                                                 bits, gs, scale, window, sinks, ws, n, None)


@pytest.mark.parametrize("status,kw", [
    (1, dict(bits=2)), (1, dict(gs=32)), (1, dict(qq=t(BF16, [3, 4, 65, 128]), parents=t(I32, [3, 65]))), (1, dict(qq=t(BF16, [3, 4, 0, 128]), parents=t(I32, [3, 0]))),
    (2, dict(qq=t(BF16, [3, 4, 128]))), (1, dict(qq=t(F32, [3, 4, 5, 128]))), (2, dict(qq=t(BF16, [3, 5, 5, 128]))), (1, dict(qq=t(BF16, [3, 4, 5, 192]), k=pool(D=192), v=pool(D=192))),
    (2, dict(res=t(BF16, [3, 4, 4, 128]))), (4, dict(res=t(F32, [3, 4, 5, 128]))), (3, dict(res=t(BF16, [3, 4, 5, 128], stride=[2560, 640, 0, 1]))),
    (2, dict(k=pool(D=64))), (2, dict(v=pool(P=5))), (1, dict(k=pool(page=24), v=pool(page=24))), (4, dict(bits=16)), (1, dict(k=pool(ptr=0x1004))),
    (2, dict(table=t(I32, [2, 4]))), (4, dict(table=t(q.INT64, [3, 4]))), (2, dict(lens=t(I32, [2]))), (2, dict(parents=t(I32, [3, 4]))), (2, dict(parents=t(I32, [2, 5]))),
    (4, dict(parents=t(q.INT64, [3, 5]))), (3, dict(parents=t(I32, [3, 5], stride=[10, 2]))), (2, dict(parents=t(I32, [15]))), (5, dict(parents=t(I32, [3, 5], ptr=None))),
    (2, dict(counts=t(I32, [2]))), (4, dict(counts=t(F32, [3]))), (2, dict(rows=t(I32, [2]))), (5, dict(scale=float("nan"))), (5, dict(scale=float("inf"))),
    (5, dict(window=-1)), (5, dict(sinks=-1)), (7, dict(ws=None)), (7, dict(n=15)), (7, dict(ws=0x1008)), (3, dict(parents=t(I32, [3, 5], ptr=0x1002))),
    (1, dict(qq=t(BF16, [1025, 4, 5, 128]), parents=t(I32, [1025, 5]), table=t(I32, [1025, 4]), lens=t(I32, [1025]))),
])
def test_tree_attention_refuses(status, kw):
    assert attend(**kw) == status, q.lib().qb200_last_error()


def test_tree_attention_of_nothing_is_nothing():
    assert attend(qq=t(BF16, [0, 4, 5, 128]), table=t(I32, [0, 4]), lens=t(I32, [0]), parents=t(I32, [0, 5])) == 0
    assert attend(qq=t(BF16, [3, 0, 5, 128])) == 0


def test_workspace_sizes():
    size = q.kv_pages_tree_attention_workspace_size
    assert size(1, 8, 2, 5, 128) >= 16
    for bad in ((0, 8, 2, 5, 128), (1, 8, 3, 5, 128), (1, 8, 2, 0, 128), (1, 8, 2, 65, 128), (1, 8, 2, 5, 96), (1, 0, 2, 5, 128), (1, 8, -1, 5, 128)):
        assert size(*bad) == 0


def accept(pools=None, table=None, lens=None, page=32, rows=NONE, parents=None, tokens=None, sampled=None, counts=NONE, path=None, nxt=None, acc=None, ends=None, n=None):
    pools = pool() if pools is None else pools
    arr = (C.POINTER(q.Tensor) * max(1, len(pools)))(*[C.pointer(p) for p in pools])
    parents = parents or t(I32, [3, 5])
    return q.lib().qb200_kv_pages_accept(*ref(path or t(I32, [3, 5]), nxt or t(I32, [3, 5]), acc or t(I32, [3]), ends or t(I32, [3])), arr, len(pools) if n is None else n,
                                         *ref(table or t(I32, [3, 4]), lens or t(I32, [3])), page, *ref(rows, parents, tokens or t(I32, [3, 5]), sampled or t(I32, [3, 5]), counts), None)


@pytest.mark.parametrize("status,kw", [
    (1, dict(page=24)), (2, dict(page=16)), (2, dict(parents=t(I32, [15]))), (1, dict(parents=t(I32, [3, 65]))), (1, dict(parents=t(I32, [3, 0]))), (2, dict(tokens=t(I32, [3, 4]))),
    (4, dict(tokens=t(q.INT64, [3, 5]))), (2, dict(sampled=t(I32, [2, 5]))), (3, dict(sampled=t(I32, [3, 5], stride=[1, 3]))), (2, dict(path=t(I32, [3, 6]))),
    (3, dict(path=t(I32, [3, 5], stride=[6, 1]))), (3, dict(nxt=t(I32, [3, 5], stride=[0, 1]))), (2, dict(acc=t(I32, [2]))), (4, dict(ends=t(F32, [3]))), (2, dict(rows=t(I32, [4]))),
    (2, dict(table=t(I32, [4, 4]), lens=t(I32, [4]))), (2, dict(lens=t(I32, [2]))), (2, dict(counts=t(I32, [1]))), (2, dict(pools=[t(BF16, [6, 2, 32])])),
    (2, dict(pools=[t(BF16, [6, 2, 32, 8]), t(BF16, [5, 2, 32, 8])])), (2, dict(pools=[t(BF16, [6, 2, 64, 8])])), (4, dict(pools=[t(q.FLOAT32 + 90, [6, 2, 32, 8])])),
    (3, dict(pools=[t(BF16, [6, 2, 32, 8], stride=[512, 0, 8, 1])])), (3, dict(pools=[t(BF16, [6, 2, 32, 8], stride=[512, 256, 4, 1])])), (5, dict(n=-1)),
    (3, dict(pools=[t(BF16, [6, 2, 32, 8], ptr=0x1001)])), (5, dict(pools=[t(BF16, [6, 2, 32, 8], ptr=None)])), (1, dict(pools=[t(BF16, [6, 1 << 17, 32, 8])])),
])
def test_accept_refuses(status, kw):
    assert accept(**kw) == status, q.lib().qb200_last_error()


def test_accept_of_no_trees_is_nothing():
    e = t(I32, [0])
    assert accept(table=t(I32, [0, 4]), lens=e, parents=t(I32, [0, 5]), tokens=t(I32, [0, 5]), sampled=t(I32, [0, 5]), path=t(I32, [0, 5]), nxt=t(I32, [0, 5]), acc=e, ends=e) == 0


def draw(logits=None, tokens=None, logprobs=NONE, random=None, temp=NONE, k=NONE, p=NONE, m=NONE):
    return q.lib().qb200_sample(*ref(tokens or t(I32, [3]), logprobs, logits or t(BF16, [3, 100]), random or t(F32, [3]), temp, k, p, m), None)


@pytest.mark.parametrize("status,kw", [
    (2, dict(logits=t(BF16, [100]))), (2, dict(logits=t(BF16, [1, 3, 100]))), (1, dict(logits=t(I32, [3, 100]))), (3, dict(logits=t(BF16, [3, 100], stride=[200, 2]))),
    (3, dict(logits=t(F32, [3, 100], ptr=0x1002))), (1, dict(logits=t(BF16, [3, 0]))), (1, dict(logits=t(BF16, [3, (1 << 19) + 1]))), (5, dict(logits=t(BF16, [3, 100], ptr=None))),
    (2, dict(random=t(F32, [2]))), (4, dict(random=t(BF16, [3]))), (2, dict(random=t(F32, [3, 1]))), (2, dict(random=NONE)), (4, dict(temp=t(F16, [3]))), (2, dict(temp=t(F32, [1]))),
    (4, dict(k=t(F32, [3]))), (2, dict(k=t(I32, [4]))), (4, dict(p=t(I32, [3]))), (4, dict(m=t(I32, [3]))), (4, dict(tokens=t(q.INT64, [3]))), (3, dict(tokens=t(I32, [3], stride=[2]))),
    (4, dict(logprobs=t(BF16, [3]))), (3, dict(logprobs=t(F32, [3], stride=[0]))), (3, dict(p=t(F32, [3], ptr=0x1001))), (5, dict(p=t(F32, [3], ptr=None))),
])
def test_sample_refuses(status, kw):
    assert draw(**kw) == status, q.lib().qb200_last_error()


def test_sample_of_no_rows_is_nothing():
    assert draw(logits=t(BF16, [0, 100]), tokens=t(I32, [0]), random=t(F32, [0])) == 0


def test_binding_takes_gpu_tensors_only():
    x, i = torch.zeros(2, 4), torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(Exception, match="CUDA tensor"):
        q.sample(x, x[:, 0])
    with pytest.raises(Exception, match="CUDA tensor"):
        q.kv_pages_accept([x], i, i[:, 0], 16, i, i, i)
    with pytest.raises(Exception, match="CUDA tensor"):
        q.kv_pages_tree_attention(x, (x, None, None), (x, None, None), i, i[:, 0], i, 16, 64, 1.0)


# ---- the restatements that the GPU tests compare with ----

def test_restated_walk_and_lines():
    parents, tokens = [-1, 0, 0, 1, 1, 3], [9, 5, 6, 5, 7, 8]
    assert walk(parents, tokens, [5, 7, 0, 0, 0, 0], 6) == [0, 1, 4]
    assert walk(parents, tokens, [5, 5, 0, 8, 0, 0], 6) == [0, 1, 3, 5]
    assert walk(parents, tokens, [5, 5, 0, 8, 0, 0], 4) == [0, 1, 3]
    assert walk(parents, tokens, [1, 5, 0, 8, 0, 0], 6) == [0] and walk(parents, tokens, [5] * 6, 0) == []
    assert line_of(parents, 5) == [5, 3, 1, 0] and line_of([3, 0, 2], 0) == [0] and line_of([3, 0, 2], 2) == [2]
    assert [j for j, _ in visible(parents, 4, 6, 10, 0, 0)] == [0, 1, 2, 3, 4, 5, 8]
    assert [j for j, _ in visible(parents, 4, 6, 10, 3, 1)] == [0, 4, 5, 8]


def test_restated_sampling():
    x = [0.0, 2.0, 1.0, 2.0]
    assert sample(x, 0.3, 0.0, 0, 1.0, 0.0)[0] == 1
    assert [sample(x, u, 1.0, 2, 1.0, 0.0)[0] for u in (0.0, 0.49, 0.51, 0.999)] == [1, 1, 3, 3]
    assert [sample(x, u, 1.0, 0, 0.3, 0.0)[0] for u in (0.0, 0.99)] == [1, 1]
    assert {sample(x, u / 100, 1.0, 0, 1.0, 0.2)[0] for u in range(100)} == {1, 2, 3}
    assert sample([float("nan"), -float("inf")], 0.5, 1.0, 0, 1.0, 0.0)[0] == -1

