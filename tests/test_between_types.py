"""What the mirror of ix_add_rms_norm, ix_kv8_append and ix_kv8_attn takes by its type: bf16 rows are bf16 tensors, not any of
two bytes."""
import pytest

import baloon_amd as bx

A = 1 << 20


def others():
    import torch
    return torch.float16, torch.int16, torch.float64


def test_norm_input():
    import torch
    t = torch.zeros
    for dtype in others():
        with pytest.raises(ValueError, match="fp32 or bf16"):
            bx.ix_add_rms_norm(1, 64, t(1, 64, dtype=dtype), None, None, t(64), 0.0, 1e-6, t(1, 64), s=0)
    assert bx.ix_add_rms_norm(1, 64, None, None, None, None, 0.0, 1e-6, None, s=0) == bx.HIP_ERROR_INVALID_VALUE


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "int16", "uint8", "float32"])
def test_rows(dtype):
    import torch
    cache = bx.kv8_cache(*(torch.zeros(s, dtype=torch.int8, device="cuda") for s in ((2, 1, 16, 64), (2, 1, 64, 16))),
                         *(torch.zeros(2, 1, device="cuda") for _ in "kv"))
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    where = (ints(0, 2), ints(2), ints(0, 1), 2)
    good, bad = (torch.ones(2, 1, 64, device="cuda").to(d) for d in (torch.bfloat16, getattr(torch, dtype)))
    o = torch.empty_like(good)
    n = bx.ix_kv8_attn_workspace_size(cache, 1, 2, 2, 1)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    attn = lambda q, gate: bx.ix_kv8_attn(cache, 1, 2, 2, *where, q, 1, 1.0, 0, 0, gate, o, ws, n)
    for call in (lambda: bx.ix_kv8_append(cache, 1, 2, *where, bad, good), lambda: bx.ix_kv8_append(cache, 1, 2, *where, good, bad),
                 lambda: attn(bad, None), lambda: attn(good, bad)):
        with pytest.raises(ValueError, match="bf16"):
            call()
    assert bx.ix_kv8_append(cache, 1, 2, *where, good, good) == 0 and attn(good, good) == 0
    assert torch.allclose(o.float(), torch.full_like(o, 0.7311, dtype=torch.float32), rtol=2 ** -7)      # sigmoid(1)
