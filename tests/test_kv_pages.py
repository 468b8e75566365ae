"""What the paged cache's entries refuse, without a GPU: through the C ABI with descriptors, and by the Python binding."""
import ctypes as C

import pytest
import torch

import qb200 as q

BF16, I32 = q.BFLOAT16, q.INT32


def t(dtype, shape, ptr=0x1000, stride=None):
    if stride is None:
        stride, acc = [], 1
        for s in reversed(shape):
            stride.insert(0, acc)
            acc *= s
    return q.raw_desc(ptr, dtype, shape, stride)


NONE = q.desc(None)


def ref(*a):
    return [None if x is None else C.byref(x) for x in a]


def pool(P=6, H=2, page=32, D=128, bits=4, **kw):
    if bits == 16:
        return [t(BF16, [P, H, page, D], **kw), NONE, NONE]
    return [t(q.UINT32, [P, H, page, D * bits // 32], **kw), t(BF16, [P, H, page, D // 64]), t(BF16, [P, H, page, D // 64])]


def append(k=None, v=None, dk=None, dv=None, table=None, rows=NONE, pos=None, counts=NONE, bits=4, gs=64):
    k, v = k or pool(), v or pool()
    dk = dk or t(BF16, [3, 2, 5, 128])
    dv = dv or dk
    return q.lib().qb200_kv_pages_append(*ref(*k, *v, dk, dv, table or t(I32, [3, 4]), rows, pos or t(I32, [3]), counts), bits, gs, None)


@pytest.mark.parametrize("status,kw", [
    (1, dict(bits=2)), (1, dict(gs=32)), (4, dict(dk=t(q.FLOAT32, [3, 2, 5, 128]))), (2, dict(dv=t(BF16, [3, 2, 4, 128]))),
    (1, dict(dk=t(BF16, [3, 2, 5, 96]))), (2, dict(k=pool(D=64))), (2, dict(v=pool(P=5))), (2, dict(k=pool(H=3))), (1, dict(k=pool(page=24), v=pool(page=24))),
    (1, dict(k=pool(page=8), v=pool(page=8))), (4, dict(bits=16)), (5, dict(bits=16, k=[pool(bits=16)[0]] + pool()[1:], v=pool(bits=16))),
    (1, dict(k=pool(ptr=0x1004))), (3, dict(k=[pool()[0], pool()[1], t(BF16, [6, 2, 32, 2], stride=[256, 128, 4, 1])])),
    (3, dict(k=[t(q.UINT32, [6, 2, 32, 16], stride=[1024, 512, 0, 1]), *pool()[1:]])), (2, dict(table=t(I32, [2, 4]))), (4, dict(table=t(q.INT64, [3, 4]))),
    (3, dict(table=t(I32, [3, 4], stride=[0, 1]))), (2, dict(pos=t(I32, [2]))), (4, dict(pos=t(q.INT64, [3]))), (2, dict(rows=t(I32, [4]))), (2, dict(counts=t(I32, [1]))),
    (3, dict(dk=t(BF16, [3, 2, 5, 128], stride=[2560, 1280, 256, 2]))), (1, dict(table=t(I32, [3, 1 << 27]))), (5, dict(dk=t(BF16, [3, 2, 5, 128], ptr=None))),
    (1, dict(dk=t(BF16, [3, 2, 1 << 30, 128], stride=[0, 0, 0, 1]))),
])
def test_append_refuses(status, kw):
    assert append(**kw) == status, q.lib().qb200_last_error()


def test_append_of_nothing_is_nothing():
    assert append(dk=t(BF16, [3, 2, 0, 128])) == 0
    assert append(dk=t(BF16, [0, 2, 5, 128]), table=t(I32, [0, 4]), pos=t(I32, [0])) == 0


def state(S=3, M=4, P=6):
    return [t(I32, [S, M]), t(I32, [S]), t(I32, [P])]


@pytest.mark.parametrize("status,st,page,n", [
    (2, [t(I32, [3, 4]), t(I32, [2]), t(I32, [6])], 32, 2), (4, [t(q.UINT32, [3, 4]), t(I32, [3]), t(I32, [6])], 32, 2), (1, state(), 33, 2), (1, state(), 0, 2),
    (1, state(P=(1 << 19) + 1), 32, 2), (5, [t(I32, [3, 4]), None, t(I32, [6])], 32, 2), (5, [t(I32, [3, 4]), t(I32, [3]), None], 32, 2), (1, state(), 32, 70000),
    (3, [t(I32, [3, 4]), t(I32, [3], stride=[2]), t(I32, [6])], 32, 2),
])
def test_bookkeeping_refuses(status, st, page, n):
    L, li = q.lib(), t(I32, [n])
    assert L.qb200_kv_pages_free(*ref(*st), page, *ref(li, NONE, NONE), None) == status
    assert L.qb200_kv_pages_fork(*ref(li, *st), page, *ref(li, li, NONE), None) == status
    assert L.qb200_kv_pages_reserve(*ref(li, t(I32, [n, 2]), *st), page, *ref(li, li), None) == status


def test_bookkeeping_refuses_lists_that_do_not_fit():
    L, st = q.lib(), state()
    two, three, pairs = t(I32, [2]), t(I32, [3]), t(I32, [2, 2])
    assert L.qb200_kv_pages_free(*ref(*st), 32, *ref(two, three, NONE), None) == 2
    assert L.qb200_kv_pages_free(*ref(*st), 32, *ref(two, NONE, three), None) == 2
    assert L.qb200_kv_pages_fork(*ref(two, *st), 32, *ref(two, three, NONE), None) == 2
    assert L.qb200_kv_pages_fork(*ref(three, *st), 32, *ref(two, two, NONE), None) == 2
    assert L.qb200_kv_pages_fork(*ref(two, *st), 32, *ref(two, two, three), None) == 2
    assert L.qb200_kv_pages_reserve(*ref(two, pairs, *st), 32, *ref(two, three), None) == 2
    assert L.qb200_kv_pages_reserve(*ref(two, t(I32, [2, 3]), *st), 32, *ref(two, two), None) == 2
    assert L.qb200_kv_pages_reserve(*ref(two, t(I32, [2, 2], stride=[4, 1]), *st), 32, *ref(two, two), None) == 2
    many = t(I32, [2049])
    assert L.qb200_kv_pages_fork(*ref(many, *st), 32, *ref(many, many, NONE), None) == 1
    assert L.qb200_kv_pages_reserve(*ref(many, t(I32, [2049, 2]), *st), 32, *ref(many, many), None) == 1
    # empty lists are done at once
    no = t(I32, [0])
    assert L.qb200_kv_pages_free(*ref(*st), 32, *ref(no, NONE, NONE), None) == 0
    assert L.qb200_kv_pages_fork(*ref(no, *st), 32, *ref(no, no, NONE), None) == 0
    assert L.qb200_kv_pages_reserve(*ref(no, t(I32, [0, 2]), *st), 32, *ref(no, no), None) == 0


def test_compact_refuses():
    L = q.lib()
    table, refs, six, one = t(I32, [3, 4]), t(I32, [6]), t(I32, [6]), t(I32, [1])
    assert L.qb200_kv_pages_compact(*ref(t(I32, [5]), t(I32, [3, 2]), one, table, refs), None) == 2
    assert L.qb200_kv_pages_compact(*ref(six, t(I32, [2, 2]), one, table, refs), None) == 2
    assert L.qb200_kv_pages_compact(*ref(six, t(I32, [3, 2]), t(I32, [2]), table, refs), None) == 2
    assert L.qb200_kv_pages_compact(*ref(six, t(I32, [3, 2], ptr=0x1004), one, table, refs), None) == 3
    assert L.qb200_kv_pages_compact(*ref(six, t(I32, [3, 2]), one, table, None), None) == 5


def copy(pools, pairs=None, count=NONE):
    arr = (C.POINTER(q.Tensor) * max(1, len(pools)))(*[C.pointer(p) for p in pools])
    return q.lib().qb200_kv_pages_copy(arr, len(pools), *ref(pairs or t(I32, [0, 2]), count), None)


@pytest.mark.parametrize("status,pools,kw", [
    (4, [t(q.INT64, [6, 4])], {}), (2, [t(BF16, [6, 4]), t(BF16, [5, 4])], {}), (2, [t(BF16, [6, 4])], dict(pairs=t(I32, [2, 3]))),
    (4, [t(BF16, [6, 4])], dict(pairs=t(q.INT64, [2, 2]))), (2, [t(BF16, [6, 4])], dict(count=t(I32, [2]))), (3, [t(BF16, [6, 4], stride=[2, 1])], {}),
    (3, [t(BF16, [6, 3, 4], stride=[64, 2, 1])], {}), (1, [t(BF16, [6, 2, 2, 2, 4], stride=[640, 200, 90, 40, 1])], {}), (5, [q.raw_desc(0x1000, BF16, [], [])], {}),
])
def test_copy_refuses(status, pools, kw):
    assert copy(pools, **kw) == status, q.lib().qb200_last_error()


def test_copy_of_nothing_is_nothing():
    assert copy([t(BF16, [6, 4])]) == 0 and copy([]) == 0 and copy([t(BF16, [6, 0, 4])], t(I32, [2, 2])) == 0


def attend(res=None, qq=None, k=None, v=None, table=None, rows=NONE, lens=None, bits=4, gs=64, window=0, sinks=0, ws=0x100000, n=1 << 30, scale=0.1):
    qq = qq or t(BF16, [3, 4, 1, 128])
    return q.lib().qb200_kv_pages_decode_attention(*ref(res or qq, qq, *(k or pool()), *(v or pool()), table or t(I32, [3, 4]), rows, lens or t(I32, [3])), bits, gs, scale,
                                                   window, sinks, ws, n, None)


@pytest.mark.parametrize("status,kw", [
    (1, dict(qq=t(q.FLOAT32, [3, 4, 1, 128]))), (2, dict(qq=t(BF16, [3, 4, 128]))), (1, dict(qq=t(BF16, [3, 4, 2, 128]))), (2, dict(res=t(BF16, [3, 4, 1, 64]))),
    (4, dict(res=t(q.FLOAT32, [3, 4, 1, 128]))), (1, dict(bits=2)), (1, dict(gs=128)), (2, dict(qq=t(BF16, [3, 5, 1, 128]))), (2, dict(k=pool(D=64))),
    (1, dict(qq=t(BF16, [3, 4, 1, 192]), k=pool(D=192), v=pool(D=192))), (2, dict(lens=t(I32, [2]))), (2, dict(table=t(I32, [4, 4]), lens=t(I32, [4]))),
    (2, dict(rows=t(I32, [2]))), (5, dict(scale=float("nan"))), (5, dict(scale=float("-inf"))), (5, dict(window=-1)), (5, dict(sinks=-1)), (7, dict(ws=None)), (7, dict(n=1024)), (7, dict(ws=0x100008)),
    (2, dict(k=pool(P=0), v=pool(P=0))), (1, dict(qq=t(BF16, [1025, 4, 1, 128]), table=t(I32, [1025, 4]), lens=t(I32, [1025]))),
    (3, dict(res=t(BF16, [3, 4, 1, 128], stride=[512, 64, 128, 1]))), (1, dict(k=pool(ptr=0x1008))), (4, dict(bits=16)),
])
def test_attention_refuses(status, kw):
    assert attend(**kw) == status, q.lib().qb200_last_error()


def test_attention_of_nothing_is_nothing():
    assert attend(qq=t(BF16, [0, 4, 1, 128]), table=t(I32, [0, 4]), lens=t(I32, [0])) == 0
    assert q.kv_pages_decode_attention_workspace_size(3, 4, 2, 128) > 0 and q.kv_pages_decode_attention_workspace_size(3, 4, 2, 96) == 0


def test_the_binding_refuses_host_tensors():
    table, lens, refs = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)
    pages = (torch.zeros(6, 2, 32, 128, dtype=torch.bfloat16), None, None)
    x = torch.zeros(3, 2, 5, 128, dtype=torch.bfloat16)
    for call in (lambda: q.kv_pages_append(pages, pages, x, x, table, lens, 16), lambda: q.kv_pages_free(table, lens, refs, 32, lens),
                 lambda: q.kv_pages_fork(table, lens, refs, 32, lens, lens), lambda: q.kv_pages_reserve(table, lens, refs, 32, lens, lens),
                 lambda: q.kv_pages_compact(table, refs), lambda: q.kv_pages_copy([pages[0]], table[:, :2].contiguous()),
                 lambda: q.kv_pages_decode_attention(x[:, :, :1], pages, pages, table, lens, 16, 64, 0.1)):
        with pytest.raises(TypeError, match="CUDA"):
            call()
    with pytest.raises(ValueError):
        q.kv_pages_append(pages[:2], pages, x, x, table, lens, 16)


@pytest.mark.parametrize("k", [
    t(q.UINT32, [6, 2, 32, 16], stride=[512, 512, 16, 1]),          # pages begin on each other's second head
    t(q.UINT32, [6, 2, 32, 16], stride=[1024, 16, 16, 1]),          # heads begin on each other's second token
    t(q.UINT32, [6, 2, 32, 16], stride=[1024, 64, 48, 1]),          # axes that are not nested
    t(q.UINT32, [6, 2, 32, 16], stride=[1 << 62, 1 << 62, 16, 1]),
])
def test_overlapping_pools_are_refused(k):
    assert append(k=[k, *pool()[1:]]) == 3, q.lib().qb200_last_error()
    assert copy([k]) in (1, 3)


def test_interleaved_pages_are_taken():
    k = t(q.UINT32, [6, 2, 32, 16], stride=[16, 6 * 16 * 32, 6 * 16, 1])       # the pages' rows lie between each other
    assert append(k=[k, *pool()[1:]], dk=t(BF16, [3, 2, 0, 128])) == 0 and copy([k]) == 0


def test_results_that_overlap_are_refused():
    assert attend(res=t(BF16, [3, 4, 1, 128], stride=[128, 128, 128, 1])) == 3
    assert q.lib().qb200_window_attention(*ref(t(BF16, [1, 2, 16, 64], stride=[0, 64, 64, 1]), *[t(BF16, [1, 2, 16, 64])] * 3), 0.1, 0, 0, *ref(NONE), None) == 3


def test_tensors_off_their_elements_are_refused():
    L, li, odd, st = q.lib(), t(I32, [2]), t(I32, [2], ptr=0x1002), state()
    assert L.qb200_kv_pages_free(*ref(*st), 32, *ref(odd, NONE, NONE), None) == 3
    assert L.qb200_kv_pages_fork(*ref(li, t(I32, [3, 4], ptr=0x1001), *st[1:]), 32, *ref(li, li, NONE), None) == 3
    assert append(dk=t(BF16, [3, 2, 5, 128], ptr=0x1001)) == 3 and append(pos=t(I32, [3], ptr=0x1002)) == 3
    assert attend(lens=t(I32, [3], ptr=0x1001)) == 3 and copy([t(BF16, [6, 4], ptr=0x1001)]) == 3


def test_a_rank_beyond_the_descriptor_is_refused():
    d = t(BF16, [6, 4])
    d.ndim = 100
    assert copy([d]) == 2
