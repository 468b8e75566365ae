"""GPU tests of the paged cache's lists: entries that reserve refuses, positions named twice, lists and pools at the launches' limits."""
import pytest
import torch

import qb200
from test_gpu_kv_pages import BF16, I32, Both, ints, make_pool, tensors

pytestmark = pytest.mark.gpu


def as_ints(t):
    return t.view(torch.int16) if t.dtype == BF16 else t


def same(got, want):
    return all(torch.equal(as_ints(a), as_ints(b)) for a, b in zip(got, want))


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_a_refused_reserve_leaves_the_cache_as_it_was(bits):
    """A full pool: a fork asks for more than there is, its new rows go to append all the same (nothing is read back), and neither its
    own rows nor those that it shares change.  The other sequence of the list is served."""
    torch.manual_seed(bits)
    page, H, D = 16, 2, 64
    st = Both(4, 6, 7, page)
    kp, vp = make_pool(7, H, page, D, bits), make_pool(7, H, page, D, bits)
    st.reserve([0, 3], [40, 30])                     # pages 0 - 2 and 3, 4
    st.fork([0], [1])
    before = [t.clone() for t in tensors(kp) + tensors(vp)]
    rows, counts = [3, 1], [2, 50]                   # the first has room; the second would take four pages of the two
    x = torch.randn(2, H, 50, D, device="cuda").to(BF16)
    pos, copies = qb200.kv_pages_reserve(st.table, st.lens, st.refs, page, ints(rows), ints(counts))
    wp, _ = st.ref.reserve(rows, counts)
    assert pos.tolist() == wp == [30, -1]
    qb200.kv_pages_copy(tensors(kp) + tensors(vp), copies)
    qb200.kv_pages_append(kp, vp, x, x, st.table, pos, bits, 64, rows=ints(rows), counts=ints(counts))
    st.check()
    want = [t.clone() for t in before]
    new = (x[0, :, :2],) if bits == 16 else qb200.quantize(x[0, :, :2].contiguous(), 64, bits)
    for w, v in zip(want, new * 2):
        w[st.ref.table[3][1], :, 14:16] = v
    assert same(tensors(kp) + tensors(vp), want)


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_a_sequence_listed_twice_is_written_once(bits):
    """The second entry is refused: its rows do not take the place of the sequence's first ones."""
    torch.manual_seed(bits)
    page, H, D, n = 16, 2, 128, 20
    st = Both(2, 6, 12, page)
    kp, vp = make_pool(12, H, page, D, bits), make_pool(12, H, page, D, bits)
    st.reserve([0], [33])
    want = [t.clone() for t in tensors(kp) + tensors(vp)]
    x = torch.randn(2, H, n, D, device="cuda").to(BF16)
    pos, _ = st.reserve([0, 0], [n, n])
    assert pos == [33, -1]
    qb200.kv_pages_append(kp, vp, x, x, st.table, ints(pos), bits, 64, rows=ints([0, 0]))
    for i in range(n):
        one = (x[0, :, i],) if bits == 16 else qb200.quantize(x[0, :, i].contiguous(), 64, bits)
        for w, v in zip(want, one * 2):
            w[st.ref.table[0][(33 + i) // page], :, (33 + i) % page] = v
    assert same(tensors(kp) + tensors(vp), want)


@pytest.mark.parametrize("bits", [4, 16])
def test_an_entry_of_a_negative_position_writes_nothing(bits):
    """However many rows it has; and a position next to 2^31 does not come around to the first ones."""
    kp, vp = make_pool(8, 2, 16, 64, bits), make_pool(8, 2, 16, 64, bits)
    before = [t.clone() for t in tensors(kp) + tensors(vp)]
    table = ints([[0, 1], [2, 3], [4, 5], [6, 7]])
    for positions, S in (([-1, -2, -3, -16], 32), ([-1, -1, -1, -1], 2), ([-2 ** 31, 2 ** 31 - 2, -2 ** 31 + 1, 2 ** 31 - 1], 40)):
        x = torch.randn(4, 2, S, 64, device="cuda").to(BF16)
        qb200.kv_pages_append(kp, vp, x, x, table, ints(positions), bits)
        qb200.kv_pages_append(kp, vp, x, x, table, ints(positions), bits, rows=ints([3, 2, 1, 0]), counts=ints([S, S, S + 9, 0]))
        assert same(tensors(kp) + tensors(vp), before)


def test_reserve_where_the_lists_take_the_last_of_the_usual_shared_memory():
    """817 entries on 131072 pages: 49108 bytes, next to the 48 KB that a launch has without asking for more."""
    st = Both(820, 3, 131072, 16)
    st.reserve([(7 * i) % 820 for i in range(817)], [i % 49 for i in range(817)])
    st.free(list(range(0, 820, 2)))
    st.reserve([(11 * i) % 820 for i in range(817)], [i % 5 for i in range(817)])


@pytest.mark.parametrize("P", [196289, 196400, 196608])
def test_compact_where_the_pages_take_the_last_of_the_usual_shared_memory(P):
    st = Both(40, 30, P, 16)
    st.reserve(list(range(40)), [(97 * i) % 480 + 1 for i in range(40)])
    st.free(list(range(0, 40, 3)))
    st.compact()
    st.refs.zero_()                                  # live pages all over the pool, a table entry for each
    st.ref.refs = [0] * P
    ids = [(i * 163 + 5) % P for i in range(1200)]
    st.table.copy_(ints(ids).view(40, 30))
    st.refs[torch.tensor(ids, device="cuda")] = 1
    st.ref.table = [ids[30 * i:30 * i + 30] for i in range(40)]
    for p in ids:
        st.ref.refs[p] = 1
    st.compact()


def test_reserve_of_a_list_that_asks_for_more_pages_than_an_int_counts():
    """17 entries of 2^27 - 1 pages each, far more than the pool has: they and the later ones that need pages are refused, those before them
    and those that need none are served."""
    S, M, P, page = 20, 2 ** 27 - 1, 64, 16
    table = torch.full((S, M), -1, dtype=I32, device="cuda")
    lens, refs = ints([0] * S), ints([0] * P)
    most = M * page - 1
    counts = [40] + [most] * 17 + [5, 0]
    pos, copies = qb200.kv_pages_reserve(table, lens, refs, page, ints(list(range(S))), ints(counts))
    assert pos.tolist() == [0] + [-1] * 18 + [0] and bool((copies == -1).all())
    assert lens.tolist() == [40] + [0] * 19 and refs.tolist() == [1] * 3 + [0] * (P - 3)
    assert table[0, :4].tolist() == [0, 1, 2, -1]
    table[0, :3] = -1
    assert all(bool((row == -1).all()) for row in table)
    assert qb200.kv_pages_reserve(table, lens, refs, page, ints([18, 19]), ints([5, 0]))[0].tolist() == [0, 0]


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_two_tokens_for_one_row_touch_no_other(bits):
    """The row holds parts of both; every other one is written or left as ever."""
    torch.manual_seed(bits)
    page, H, D = 16, 3, 128
    kp, vp = make_pool(6, H, page, D, bits), make_pool(6, H, page, D, bits)
    want = [t.clone() for t in tensors(kp) + tensors(vp)]
    x = torch.randn(3, H, 2, D, device="cuda").to(BF16)
    qb200.kv_pages_append(kp, vp, x, x, ints([[2, 4], [5, 4]]), ints([15, 7, 16]), bits, rows=ints([0, 1, 1]))      # (0, 16) and (1, 16) are one row
    new = (x,) if bits == 16 else qb200.quantize(x, 64, bits)
    for w, t, v in zip(want, tensors(kp) + tensors(vp), new * 2):
        w[2, :, 15], w[5, :, 7], w[5, :, 8], w[4, :, 1] = v[0, :, 0], v[1, :, 0], v[1, :, 1], v[2, :, 1]
        row, one, two = as_ints(t[4, :, 0]), as_ints(v[0, :, 1]), as_ints(v[2, :, 0])
        assert bool(((row == one) | (row == two)).all())
        w[4, :, 0] = t[4, :, 0]
    assert same(tensors(kp) + tensors(vp), want)
