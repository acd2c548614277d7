"""Which attention AttnLayer takes for slots that were forked from one prompt, and the hybrid stack with either."""
import pytest

import baloon_amd as bx
import baloon_amd.layer
from tests.test_attn_layer_fork import check, drawn
from tests.test_kv8_cache import cumulative, ints

pytestmark = pytest.mark.gpu


@pytest.fixture
def taken(monkeypatch):
    """The attention calls that were made, by name and groups."""
    made = []
    for name in ("ix_kv8_attn", "ix_kv8_attn_shared"):
        def call(*args, name=name, real=getattr(bx, name)):
            made.append((name, args[8] if name == "ix_kv8_attn_shared" else 0))
            return real(*args)
        monkeypatch.setattr(baloon_amd.layer, name, call)

    def last():
        got = made[:]
        made.clear()
        return got
    return last


ALONE, SHARED = [("ix_kv8_attn", 0)], [("ix_kv8_attn_shared", 1)]


@pytest.mark.parametrize("more", [-1, 0, 1])
def test_worth(taken, more):
    """3 slots behind 100 tokens spare 200 tokens of 2 heads of 64 channels: 25,600 codes."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(1)
    layer = bx.AttnLayer(4, 300, 4, 2, 64, 16, max_forks=1, worth=25600 + more)

    def step(*lens):
        rows = drawn(g, sum(lens), 4, 2, 64)
        got = layer.decode(*rows) if lens == (1,) * 4 else layer.prefill(ints(cumulative(lens)), max(lens), *rows)
        check(layer, lens, rows[0], rows[3], got)

    step(100, 0, 0, 7)
    assert taken() == ALONE
    layer.fork(0, 3, 100)
    step(1, 1, 1, 1)
    assert taken() == (ALONE if more > 0 else SHARED)
    layer.release(0)
    step(1, 1, 1, 1)
    assert taken() == ALONE


def test_how_many_tokens(taken):
    """Calls of up to 16 tokens a slot in the mean, however they are spread."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(2)
    layer = bx.AttnLayer(4, 700, 4, 2, 64, 16, max_forks=2, worth=0)

    def step(*lens):
        rows = drawn(g, sum(lens), 4, 2, 64)
        got = layer.prefill(ints(cumulative(lens)), max(lens), *rows)
        check(layer, lens, rows[0], rows[3], got)

    step(100, 0, 0, 7)
    layer.fork(0, 3, 100)
    taken()
    for lens, want in (((16, 16, 16, 16), SHARED), ((17, 16, 16, 16), ALONE), ((0, 64, 0, 0), SHARED), ((0, 65, 0, 0), ALONE), ((0, 0, 0, 64), SHARED),
                       ((1, 0, 0, 0), SHARED)):
        step(*lens)
        assert taken() == want, lens


def test_two_forks_and_what_lies_between(taken):
    """Groups side by side: two forks, and one between them that shares nothing; what they spare is added up."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(3)
    layer = bx.AttnLayer(8, 300, 4, 2, 64, 16, max_forks=2, worth=(100 + 2 * 50) * 128)
    lens = (100, 0, 3, 3, 50, 0, 0, 9)
    layer.prefill(ints(cumulative(lens)), 100, *drawn(g, sum(lens), 4, 2, 64))
    layer.fork(0, 2, 100)
    rows = drawn(g, 8, 4, 2, 64)
    check(layer, [1] * 8, rows[0], rows[3], layer.decode(*rows))
    layer.fork(4, 3, 50)
    taken()
    rows = drawn(g, 8, 4, 2, 64)
    check(layer, [1] * 8, rows[0], rows[3], layer.decode(*rows))
    assert taken() == [("ix_kv8_attn_shared", 3)]
    assert layer._groups.tolist() == [0, 2, 4, 7, 7] and layer._shared.tolist() == [100, 0, 50, 0]


@pytest.mark.parametrize("worth", [0, 200_000_000])
def test_continuations(taken, worth):
    """The hybrid stack's continuations by either attention end where a pass over their tokens ends, within what
    tests/test_attn_layer.py derives for tokens against one prompt."""
    import torch
    from examples import hybrid
    prompts = [[i % 512 for i in range(5, 305)], [1, 2, 3], list(range(64))]
    made, model = hybrid.continuations(prompts, 2, 6, worth=worth)
    names = [name for name, _ in taken()]
    assert names == ["ix_kv8_attn"] + ["ix_kv8_attn" if worth else "ix_kv8_attn_shared"] * 6
    whole = hybrid.Hybrid(6, 400, rope_base=1e4)
    tokens = [prompts[i // 2] + m for i, m in enumerate(made)]
    lens = [len(t) for t in tokens]
    whole.forward(torch.tensor(sum(tokens, []), device="cuda"), ints(cumulative(lens)), max(lens))
    a, b = model.hidden_state.double(), whole.hidden_state.double()
    assert torch.isfinite(a).all()
    assert ((a - b).norm(dim=1) <= 0.125 * b.norm(dim=1)).all(), ((a - b).norm(dim=1) / b.norm(dim=1)).tolist()
