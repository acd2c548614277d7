"""AttnLayer against the plain attention over its own cache, and the hybrid stack of examples/hybrid.py."""
import numpy as np
import pytest

import baloon_amd as bx
from tests import kv8_ref
from tests.test_kv8_cache import bf, cumulative, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("own_pages", [True, False])
@pytest.mark.parametrize("window,sinks", [(0, 0), (48, 3)])
def test_prompts_drafts_tokens(own_pages, window, sinks):
    """Prompts, single tokens, a dropped draft and more tokens: after each the output is the attention over the cache's
    values (read back by ix_kv8_read), and those are the rows appended to within a page's scale / 2, twice rounded.

    Output tolerance: as in the kernel's own test at these sizes, 2^-8 of the result and 2^-9 of the largest value."""
    import torch
    n, h_q, h_kv, d, page = 3, 4, 2, 64, 32
    layer = bx.AttnLayer(n, 300, h_q, h_kv, d, page, None if own_pages else 40, window, sinks)
    if not own_pages:
        layer.table.copy_(torch.randperm(40)[:30].view(3, 10))
    g = np.random.default_rng(0)
    held = [np.zeros((2, 0, h_kv, d)) for _ in range(n)]
    length = np.zeros(n, int)
    for step, lens in enumerate([(37, 5, 200), (1, 1, 1), (4, 4, 4), "drop", (1, 1, 1), (0, 50, 2)]):
        if lens == "drop":
            layer.kv_len -= 3
            length -= 3
            held = [x[:, :m] for x, m in zip(held, length)]
            continue
        T = sum(lens)
        (qb, q), (zb, z) = (kv8_ref.normal_bf16(g, T, h_q, d) for _ in "qz")
        (kb, k), (vb, v) = (kv8_ref.normal_bf16(g, T, h_kv, d) for _ in "kv")
        if lens == (1, 1, 1):
            got = layer.decode(bf(qb), bf(kb), bf(vb), bf(zb))
        else:
            got = layer.prefill(ints(cumulative(lens)), max(lens), bf(qb), bf(kb), bf(vb), bf(zb))
        got = got.float().cpu().numpy()
        cu = cumulative(lens)
        length += lens
        assert layer.kv_len.tolist() == length.tolist()
        all_k, all_v = (torch.empty(length.sum(), h_kv, d, dtype=torch.bfloat16, device="cuda") for _ in "kv")
        assert bx.ix_kv8_read(layer.cache, n, int(length.sum()), ints(cumulative(length)), layer.kv_len, layer.table, layer.width,
                              all_k, all_v) == 0
        t = layer.cache.tensors
        ids, at = layer.table.cpu().numpy(), 0
        for b, m in enumerate(lens):
            held[b] = np.concatenate([held[b], np.stack([k, v])[:, cu[b]:cu[b + 1]]], 1)
            tokens = np.arange(length[b])
            codes = [t[0].cpu().numpy()[ids[b, tokens // page], :, tokens % page],
                     t[1].cpu().numpy()[ids[b, tokens // page], :, :, tokens % page]]
            scales = [t[2 + i].cpu().numpy()[ids[b, tokens // page]][:, :, None] for i in range(2)]
            for i in range(2):
                value = codes[i].astype(np.float64) * scales[i]
                assert np.all(np.abs(value - held[b][i]) <= 1.01 * scales[i] * (0.5 + 0.5 * (step + 1)))     # one more half a rescaling
                read = (all_k, all_v)[i][at:at + length[b]].float().cpu().numpy()
                assert np.all(np.abs(read - value) <= 2.0 ** -8 * np.abs(value))
            at += length[b]
            ones = np.ones(length[b], bool)
            seen = kv8_ref.seen_by(m, length[b], ones, window, sinks)
            kk, vv = (codes[i].astype(np.float64) * scales[i] for i in range(2))
            want = kv8_ref.attend(q[cu[b]:cu[b + 1]], length[b], kk, vv, seen, layer.scale, z[cu[b]:cu[b + 1]])
            assert np.all(np.abs(got[cu[b]:cu[b + 1]] - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -9 * (np.abs(vv).max() if m else 0))


def test_refusals():
    import torch
    layer = bx.AttnLayer(2, 64, 4, 2, 64, 16)
    q, k = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: layer.decode(q[:1], k[:1], k[:1]), lambda: layer.decode(q, k[:1], k), lambda: layer.decode(q, k, k, q[:1]),
                 lambda: layer.prefill(ints([0, 2]), 2, q, k, k)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(bx.IxGdnError):
        layer.prefill(ints([0, 1, 2]), 0, q, k, k)              # no new tokens at most
    assert layer.kv_len.tolist() == [0, 0]
    with pytest.raises(bx.IxGdnError):
        bx.AttnLayer(2, 64, 5, 2, 64, 16).decode(torch.zeros(2, 5, 64, dtype=torch.bfloat16, device="cuda"), k, k)


def test_hybrid_stack():
    """Generated token by token, the stack ends where one prompt of all the tokens ends. The two differ by roundings of the
    layers' bf16 outputs and of pages' scales that grow in different steps, 2^-9 and 2^-8 of a value each over 4 layers of
    about 8 roundings: in all below 32 * 2^-8, a part of 0.125 of the norm, if every one of them pointed the same way."""
    import torch
    from examples import hybrid
    prompts = [[i % 512 for i in range(5, 305)], [1, 2, 3], list(range(64))]
    made, model = hybrid.generate(prompts, 6)
    assert len(made) == 3 and all(len(m) == 6 for m in made)
    whole = hybrid.Hybrid(3, 400)
    lens = [len(p) + 6 for p in prompts]
    whole.forward(torch.tensor(sum((p + m for p, m in zip(prompts, made)), []), device="cuda"), ints(cumulative(lens)), max(lens))
    a, b = model.hidden_state.double(), whole.hidden_state.double()
    assert torch.isfinite(a).all()
    assert ((a - b).norm(dim=1) <= 0.125 * b.norm(dim=1)).all(), ((a - b).norm(dim=1) / b.norm(dim=1)).tolist()
