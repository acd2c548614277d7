"""Calls without tokens or rows: the addresses of tensors without elements are 0, and nothing is done."""
import pytest

import baloon_amd as bx
from tests.test_add_norm import call as norm
from tests.test_kv8_attn import attn
from tests.test_kv8_cache import append, desc, read

INVALID = bx.HIP_ERROR_INVALID_VALUE


def test_no_rows():
    assert norm(rows=0, x=None, res=None, res_out=None, w=None, y=None) == bx.HIP_SUCCESS
    assert norm(rows=0, n=0) == INVALID and norm(rows=0, n=48, q=1 << 20) == INVALID
    assert append(T=0, k=(None, 128), v=(None, 128)) == bx.HIP_SUCCESS
    assert read(T=0, k=None, v=None) == bx.HIP_SUCCESS
    assert attn(T=0, max_q=0, q=(None, 256), gate=(None, 256), o=None) == bx.HIP_SUCCESS
    for f in (append, read, attn):                              # a batch and a cache they are all the same
        assert f(desc(page=48), T=0) == INVALID and f(T=0, n_seq=0) == INVALID and f(T=0, cu=None) == INVALID
    assert attn(T=0, h_q=3) == INVALID


@pytest.mark.gpu
def test_tensors_without_elements():
    import torch
    rows, w = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(128, device="cuda")
    assert bx.ix_add_rms_norm(0, 128, rows, rows, rows, w, 0.0, 1e-6, None, rows) == 0
    layer = bx.AttnLayer(2, 64, 2, 2, 64, 16)
    layer.kv_len.copy_(torch.tensor([3, 0], dtype=torch.int32))
    o = layer.prefill(torch.zeros(3, dtype=torch.int32, device="cuda"), 0, rows, rows, rows)
    assert o.shape == (0, 2, 64) and layer.kv_len.tolist() == [3, 0]
    where = (layer.cache, 2, 0, torch.zeros(3, dtype=torch.int32, device="cuda"), layer.kv_len, layer.table, layer.width)
    assert bx.ix_kv8_read(*where, rows, rows) == 0
