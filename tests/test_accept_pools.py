"""A list of pools whose rows move may name none of them twice: rows that have moved would move again."""
import pytest

import qb200 as q
from test_drafted import accept
from test_kv_pages import BF16, I32, t


def pools(*starts):
    return [t(BF16, [6, 2, 32, 8], ptr=p) for p in starts]


@pytest.mark.parametrize("starts", [(0x10000, 0x10000), (0x10000, 0x20000, 0x30000, 0x20000), tuple(range(0x100000, 0x100000 + 300 * 4096, 4096)) + (0x100000,)])
def test_a_pool_listed_twice_is_refused(starts):
    assert accept(pools=pools(*starts)) == 5 and b"twice" in q.lib().qb200_last_error()


def test_no_trees_move_nothing():
    e, i = t(I32, [0]), t(I32, [0, 5])
    for P in (0, 6):
        two = [t(BF16, [P, 2, 32, 8]), t(BF16, [P, 2, 32, 8])]
        assert accept(pools=two, table=t(I32, [0, 4]), lens=e, parents=i, tokens=i, sampled=i, path=i, nxt=i, acc=e, ends=e) == 0
