"""Many empty groups, as a captured call may have for later: they take no room."""
import pytest

import baloon_amd as bx
from tests.test_kv8_cache import desc
from tests.test_kv8_shared import Shared, group


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n_seq,T", [(64, 64), (5, 5), (64, 3), (1, 7), (300, 9000)])
def test_workspace(d, n_seq, T):
    """A group with rows has two sequences or more and a token: more groups than those need no more workspace."""
    sizes = [bx.ix_kv8_attn_shared_workspace_size(desc(d=d, h=2), n_seq, T, T, n, 16) for n in (1, 2, 30, min(n_seq // 2, T) or 1, 400, 65535)]
    assert 0 < sizes[0] and sizes[-1] == sizes[-2] == max(sizes)
    assert sizes[3] == sizes[-1]


@pytest.mark.gpu
@pytest.mark.parametrize("page,h,d,G", [(16, 3, 64, 2), (64, 1, 256, 8), (32, 5, 128, 4)])
def test_pairs(page, h, d, G):
    """As many groups with rows as there can be, and empty ones before, between and behind: the room is full."""
    for n in (1, 40):
        for tokens in (70, 700):
            groups = []
            for i in range(n):
                groups += [group(0)] * (i % 3) + [group(tokens, (1, 1 + i % 5), (i % 2, 2 + i % 7))]
            Shared(groups + [group(0)] * 100, page=page, h=h, d=d, G=G, seed=n).both()


@pytest.mark.gpu
def test_blocks_of_pairs():
    """The same by blocks of 128 rows, a few more rows than a block holds in each group."""
    p = Shared([group(0)] * 5 + [group(3000, (3, 3), (2, 9)) for _ in range(20)] + [group(0)] * 5, page=128, h=3, d=64, G=27)
    p.both()
