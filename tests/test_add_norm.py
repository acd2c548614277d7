"""ix_add_rms_norm: h = bf16(x + res), y = h / sqrt(mean(h^2) + eps) * (w0 + w).

The stream h is compared bit for bit, y against the formula in 64 bits on that h. The kernel sums at most 32
squares in a thread one after another and 16 + 16 more partial sums in a tree, so the sum of squares (all
terms positive) is within 64 * 2^-24 of its value, the inverse root within half of that, and the division,
root and three products add under 6 * 2^-24: 40 * 2^-24 = 2.4e-6 relative. A bf16 output adds half a bf16 ulp. q8_1
blocks equal ix_q8_1_quantize's of the fp32 output byte for byte."""
import ctypes

import numpy as np
import pytest

import baloon_amd as bx
from oracle import bf16

INVALID = bx.HIP_ERROR_INVALID_VALUE
REL = 40 * 2.0 ** -24
A = 1 << 20


def call(rows=2, n=64, x=A, x16=None, res=A, res_out=A, w=A, y=A, y16=None, q=None):
    f = ctypes.c_float
    return bx.lib().ix_add_rms_norm(rows, n, x, x16, res, res_out, w, f(0), f(1e-6), y, y16, q, None)


def test_refusals():
    assert call(rows=-1) == INVALID
    assert call(n=0) == INVALID and call(n=-8) == INVALID and call(n=32769) == INVALID
    assert call(x=None) == INVALID and call(x16=A) == INVALID            # one input, not none and not two
    assert call(w=None) == INVALID
    assert call(y=None) == INVALID                                       # nothing to write
    assert call(n=48, q=A) == INVALID                                    # not whole q8_1 blocks
    for odd in (dict(x=A + 2), dict(x=None, x16=A + 1), dict(res=A + 1), dict(res_out=A + 1), dict(w=A + 2), dict(y=A + 2),
                dict(y16=A + 1), dict(q=A + 2)):
        assert call(**odd) == INVALID, odd
    assert call(rows=0) == bx.HIP_SUCCESS                                # no rows: no launch


def expected(x, res, w, w0, eps):
    """(h bits, y in 64 bits)"""
    h = bf16.from_f32(x + bf16.to_f32(res) if res is not None else x)
    z = bf16.to_f32(h).astype(np.float64)
    return h, z / np.sqrt((z * z).mean(1, keepdims=True) + eps) * (w0 + w.astype(np.float64))


def data(rows, n, seed):
    g = np.random.default_rng(seed)
    x = g.normal(0, 1, (rows, n)).astype(np.float32)
    return x, bf16.from_f32(g.normal(0, 2, (rows, n)).astype(np.float32)), g.normal(0, 0.2, n).astype(np.float32)


def dev(a):
    import torch
    a = np.ascontiguousarray(a)
    if a.dtype == np.uint16:
        return torch.from_numpy(a.view(np.int16).copy()).view(torch.bfloat16).cuda()
    return torch.from_numpy(a.copy()).cuda()


def bits(t):
    import torch
    return t.cpu().view(torch.int16).numpy().view(np.uint16)


def check_y(got, want, rel=REL):
    assert np.all(np.abs(got.astype(np.float64) - want) <= rel * np.abs(want) + 1e-30)


SIZES = [(1, 1), (3, 7), (1, 8), (2, 32), (5, 500), (1, 513), (2, 1000), (1, 2048), (7, 2048), (3, 2049), (2, 4096),
         (1, 4104), (2, 5000), (1, 8192), (2, 8200), (1, 20000), (1, 32768), (1, 32767), (1500, 96), (1030, 2048),
         (1025, 4096)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", SIZES)
@pytest.mark.parametrize("fp32", [False, True])
def test_against_64_bits(rows, n, fp32):
    import torch
    x, res, w = data(rows, n, rows * 40000 + n)
    if not fp32:
        x = bf16.to_f32(bf16.from_f32(x))
    h_want, y_want = expected(x, res, w, 1.0, 1e-6)
    tx = dev(x) if fp32 else dev(bf16.from_f32(x))
    tr = dev(res)
    y = torch.full((rows, n), float("nan"), device="cuda")
    y16 = torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda")
    q = torch.full((rows * n // 32, 36), 0xAA, dtype=torch.uint8, device="cuda") if n % 32 == 0 else None
    assert bx.ix_add_rms_norm(rows, n, tx, tr, tr, dev(w), 1.0, 1e-6, y, y16, q) == 0
    assert np.array_equal(bits(tr), h_want)                              # in place
    got = y.cpu().numpy()
    check_y(got, y_want)
    assert np.array_equal(bits(y16), bf16.from_f32(got))
    if q is not None:
        q2 = torch.zeros_like(q)
        assert bx.ix_q8_1_quantize(y, q2, rows * n) == 0
        assert torch.equal(q, q2)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [40, 2048, 2050])
def test_operands(n):
    """Without a residual, one output at a time, outputs over inputs, operands off a 16-byte line."""
    import torch
    rows = 5
    x, res, w = data(rows, n, n)
    x16 = bf16.from_f32(x)
    x = bf16.to_f32(x16)
    tw = dev(w)
    h_want, y_want = expected(x, None, w, 0.0, 1e-5)
    y = torch.empty(rows, n, device="cuda")
    assert bx.ix_add_rms_norm(rows, n, dev(x16), None, None, tw, 0.0, 1e-5, y) == 0
    check_y(y.cpu().numpy(), y_want)
    h_want, y_want = expected(x, res, w, 0.0, 1e-5)
    y32 = torch.empty(rows, n, device="cuda")
    assert bx.ix_add_rms_norm(rows, n, dev(x16), dev(res), None, tw, 0.0, 1e-5, y32) == 0
    want16 = bf16.from_f32(y32.cpu().numpy())
    check_y(y32.cpu().numpy(), y_want)
    tx, out = dev(x16), dev(res)
    assert bx.ix_add_rms_norm(rows, n, tx, out, out, tw, 0.0, 1e-5, None, tx) == 0        # y over x, h over res
    assert np.array_equal(bits(tx), want16) and np.array_equal(bits(out), h_want)
    tx, tr = dev(x16), dev(res)
    assert bx.ix_add_rms_norm(rows, n, tx, tr, tx, tw, 0.0, 1e-5, None, tr) == 0          # h over x, y over res
    assert np.array_equal(bits(tr), want16) and np.array_equal(bits(tx), h_want)
    off = torch.empty(rows * n + 1, dtype=torch.bfloat16, device="cuda")[1:]
    off.copy_(dev(x16).view(-1))
    y2 = torch.empty(rows, n, device="cuda")
    assert bx.ix_add_rms_norm(rows, n, off, dev(res), None, tw, 0.0, 1e-5, y2) == 0
    check_y(y2.cpu().numpy(), y_want)


@pytest.mark.gpu
def test_rows_of_zeros_and_large_values():
    import torch
    n = 256
    x = np.zeros((4, n), np.float32)
    x[1] = 1e18                                               # squares of 1e36, whose sum is still finite in 32 bits
    x[2, 5] = np.inf
    x[3] = 1e-30                                              # squares under the smallest float: eps decides
    w = np.ones(n, np.float32)
    y = torch.empty(4, n, device="cuda")
    assert bx.ix_add_rms_norm(4, n, dev(x), None, None, dev(w), 0.0, 1e-6, y) == 0
    got = y.cpu().numpy()
    assert np.all(got[0] == 0)
    assert np.allclose(got[1], 1, rtol=REL)
    assert np.isnan(got[2, 5]) and np.all(got[2, :5] == 0)    # inf / inf, 0 / inf: the row alone
    h = bf16.to_f32(bf16.from_f32(x[3]))
    assert np.allclose(got[3], h * 1e3, rtol=1e-5, atol=0)


@pytest.mark.gpu
def test_stream_and_graph():
    """On another stream than the tensors' own, and captured: every replay equals the eager call."""
    import torch
    rows, n = 3, 2048
    x, res, w = data(rows, n, 9)
    tx, tr, tw = dev(bf16.from_f32(x)), dev(res), dev(w)
    y, h = (torch.empty(rows, n, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    assert bx.ix_add_rms_norm(rows, n, tx, tr, h, tw, 0.0, 1e-6, None, y) == 0
    torch.cuda.synchronize()
    want = bits(y).copy()
    side = torch.cuda.Stream()
    y.zero_()
    side.wait_stream(torch.cuda.current_stream())
    assert bx.ix_add_rms_norm(rows, n, tx, tr, h, tw, 0.0, 1e-6, None, y, None, side) == 0
    side.synchronize()
    assert np.array_equal(bits(y), want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        assert bx.ix_add_rms_norm(rows, n, tx, tr, h, tw, 0.0, 1e-6, None, y) == 0
    for _ in range(3):
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(bits(y), want)
