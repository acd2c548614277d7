"""ix_kv8_append_rope's queries: in the append's own launch where that has the waves for them, else in one of their own; the same
bits on both sides of the limit."""
import pytest

import baloon_amd as bx
from tests import launches
from tests.test_kv8_cache import Pair, ints, tables_for
from tests.test_rope import append_both, make

pytestmark = pytest.mark.gpu


def call_of(h_q, h_kv, d, page, n_seq, each):
    import torch
    T, width = n_seq * each, -(-each // page)
    n = n_seq * width
    cache = bx.kv8_cache(torch.zeros(n, h_kv, page, d, dtype=torch.int8, device="cuda"), torch.zeros(n, h_kv, d, page, dtype=torch.int8, device="cuda"),
                         torch.zeros(n, h_kv, device="cuda"), torch.zeros(n, h_kv, device="cuda"))
    r = bx.rope(bx.rope_freq(d)[0].cuda())
    q, k, v = (torch.zeros(T, h, d, dtype=torch.bfloat16, device="cuda") for h in (h_q, h_kv, h_kv))
    a = (cache, n_seq, T, ints(range(0, T + 1, each)), ints([each] * n_seq), ints(range(n)).view(n_seq, width), width, k, v, r, q, h_q, r,
         torch.empty_like(q))

    def call(s=None):
        assert bx.ix_kv8_append_rope(*a, s) == 0
    call()
    return call


@pytest.mark.parametrize("h_q,h_kv,d,page,n_seq,each,want", [
    (16, 1, 256, 128, 1, 1024, 2), (64, 1, 64, 128, 1, 1024, 2), (16, 2, 256, 64, 1, 1024, 2), (32, 1, 128, 16, 1, 600, 2),
    (16, 2, 256, 16, 64, 1, 1), (32, 8, 128, 32, 37, 4, 1), (16, 1, 128, 64, 64, 1, 1), (64, 1, 256, 64, 16, 1, 1), (16, 2, 256, 64, 1, 1, 1)])
def test_where_the_queries_go(h_q, h_kv, d, page, n_seq, each, want):
    assert launches.count(call_of(h_q, h_kv, d, page, n_seq, each)) == want


@pytest.mark.parametrize("page,h,d,G,lens", [(128, 1, 256, 16, [1024]), (128, 1, 64, 64, [1000, 3]), (64, 2, 256, 8, [700, 1, 324]), (16, 1, 128, 32, [600]),
                                             (128, 1, 128, 32, [20]), (128, 1, 128, 32, [70])])
def test_few_pages(page, h, d, G, lens):
    """Prompts whose pages are few beside their queries."""
    width = max(lens) // page + 2
    p = Pair(len(lens) * width, page, h, d, page + d + G)
    tables = tables_for(p.g, len(lens) * width, [n + 1 for n in lens], page, width)
    (rk, _), (rq, _) = make(p.g, d, d // 2), make(p.g, d, d, 1, False)
    append_both(p, lens, list(lens), tables, G * h, rk, rq)
    append_both(p, [1] * len(lens), [n + 1 for n in lens], tables, G * h, rk, rq)
