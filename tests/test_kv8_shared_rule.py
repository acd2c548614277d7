"""Which kernels ix_kv8_attn_shared may take where one of its groups has most of the rows."""
import pytest

import baloon_amd as bx
from tests import launches
from tests.test_kv8_cache import ints
from tests.test_kv8_shared import Shared, group

pytestmark = pytest.mark.gpu


def call_of(n, shared, n_groups, d, h, G):
    """(call, keep): n sequences of a token behind `shared` ones, the first of n_groups groups; the others are empty."""
    import torch
    page = 128
    pages = shared // page + 1
    cache = bx.kv8_cache(torch.zeros(pages, h, page, d, dtype=torch.int8, device="cuda"), torch.zeros(pages, h, d, page, dtype=torch.int8, device="cuda"),
                         torch.ones(pages, h, device="cuda"), torch.ones(pages, h, device="cuda"))
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(n, 1)
    q = torch.zeros(n, h * G, d, dtype=torch.bfloat16, device="cuda")
    o = torch.empty_like(q)
    need = bx.ix_kv8_attn_shared_workspace_size(cache, n, n, 1, n_groups, h * G)
    a = (cache, n, n, 1, ints(range(n + 1)), ints([shared + 1] * n), table, pages, n_groups, ints([0] + [n] * n_groups), ints([shared] + [0] * (n_groups - 1)),
         q, h * G, 1.0, None, o, torch.empty(need, dtype=torch.uint8, device="cuda"), need)

    def call(s=None):
        assert bx.ix_kv8_attn_shared(*a, s) == 0
    call()
    return call


@pytest.mark.parametrize("n,shared,n_groups,d,h,G,want", [
    (128, 16384, 1, 256, 2, 8, 3), (128, 16384, 64, 256, 2, 8, 3), (256, 16384, 64, 256, 2, 8, 3), (96, 16384, 20, 128, 8, 4, 3),
    (4, 16384, 1, 256, 2, 8, 2), (64, 2048, 64, 256, 2, 8, 2), (128, 100, 64, 64, 1, 1, 2)])
def test_one_large_group(n, shared, n_groups, d, h, G, want):
    """A group whose tiles are many is open to the kernel of 128 rows, however many empty ones there are beside it: a launch more
    than where no group can have that many."""
    assert launches.count(call_of(n, shared, n_groups, d, h, G)) == want


@pytest.mark.parametrize("d,h,G,n", [(64, 2, 16, 20), (128, 4, 4, 40), (256, 2, 8, 20)])
@pytest.mark.parametrize("at", [0, 40])
def test_one_large_group_among_small_ones(d, h, G, n, at):
    """n sequences of 4 new tokens behind 9,000 among 63 groups of two and of none."""
    small = [group(40, (1, 3), (1, 5)) if i % 3 == 0 else group(0) for i in range(63)]
    Shared(small[:at] + [group(9000, *[(4, 4 + i % 7) for i in range(n)])] + small[at:], page=64, h=h, d=d, G=G).both()
