"""GdnLayer and AttnLayer: device-resident parameters and per-sequence states of one layer.

GdnLayer is a thin host object over the C ABI: it owns the conv weights, A_log, dt_bias, the recurrent
state block [n][h_v][d_v][d_k] fp32 (each head's state stored column by column), the conv
state [n][C][d_conv-1] bf16, the gated output norm's weight ssm_norm [d_v] fp32 and the
zeroed decode workspace, and calls ``ix_gdn_decode`` / ``ix_gdn_prefill`` (or their gated
variants, when a gate input z is passed) on the current stream. Allocation happens here, at
construction (and for the prefill workspace, on first use of a given size), never inside the
library calls.

AttnLayer is the same for the softmax attention layers that stand between GDN layers: it owns a paged 8-bit
cache of keys and values and the lengths of its sequences, and calls ``ix_kv8_append`` and ``ix_kv8_attn``.
"""
from __future__ import annotations

import torch

from . import (HIP_ERROR_INVALID_VALUE, Cfg, _rows, check, ix_gdn_decode, ix_gdn_decode_gated, ix_gdn_decode_workspace_size, ix_gdn_prefill,
               ix_gdn_prefill_gated, ix_gdn_prefill_gated_workspace_size, ix_gdn_prefill_workspace_size,
               ix_kv8_append, ix_kv8_attn, ix_kv8_attn_workspace_size, kv8_cache, make_cfg, out_gate)


class GdnLayer:
    def __init__(self, n_slots: int, cfg: Cfg | None = None, device="cuda"):
        self.cfg = cfg or make_cfg()
        c = self.cfg
        self.n_slots = n_slots
        self.device = torch.device(device)
        C = c.channels
        self.conv_w = torch.zeros(C, c.d_conv, dtype=torch.bfloat16, device=self.device)
        self.A_log = torch.zeros(c.h_v, dtype=torch.float32, device=self.device)
        self.dt_bias = torch.zeros(c.h_v, dtype=torch.float32, device=self.device)
        self.state = torch.zeros(n_slots, c.h_v, c.d_v, c.d_k, dtype=torch.float32, device=self.device)
        self.conv_state = torch.zeros(n_slots, C, c.d_conv - 1, dtype=torch.bfloat16, device=self.device)
        self.ssm_norm = torch.ones(c.d_v, dtype=torch.float32, device=self.device)
        self.norm_eps = 1e-6
        self.decode_ws = torch.zeros(ix_gdn_decode_workspace_size(c, n_slots), dtype=torch.uint8, device=self.device)
        self._ws = None

    def decode(self, x, a, b, o=None, o_bf16=None, z=None, y=None, y_bf16=None, y_q8_1=None, stream=None):
        """One token for all n_slots sequences: x [n][C] bf16, a, b [n][h_v] bf16. With z
        [n][h_v][d_v] bf16 the gated output norm is fused in and written to y, y_bf16 and/or
        y_q8_1 (uint8, 36 bytes per 32 outputs: the activation format of ix_mmvq_q8_0)."""
        args = (self.cfg, self.n_slots, x, self.conv_state, self.conv_w, a, b, self.A_log, self.dt_bias, self.state,
                o, o_bf16)
        if z is None:
            check("ix_gdn_decode", ix_gdn_decode(*args, self.decode_ws, stream))
        else:
            g = out_gate(z, self.ssm_norm, self.norm_eps, y, y_bf16, y_q8_1)
            check("ix_gdn_decode_gated", ix_gdn_decode_gated(*args, g, self.decode_ws, stream))

    def prefill(self, cu_seqlens, x, a, b, o=None, o_bf16=None, z=None, y=None, y_bf16=None, y_q8_1=None,
                stream=None):
        """Packed prefill of n_slots sequences (cu_seqlens int32 [n+1] on the device); z, y,
        y_bf16, y_q8_1 as in decode, with [total_T] rows."""
        total_T = x.shape[0]
        size = ix_gdn_prefill_workspace_size if z is None else ix_gdn_prefill_gated_workspace_size
        need = size(self.cfg, self.n_slots, total_T)
        if self._ws is None or self._ws.numel() < need:
            self._ws = torch.empty(max(need, 256), dtype=torch.uint8, device=self.device)
        args = (self.cfg, self.n_slots, total_T, cu_seqlens, x, self.conv_state, self.conv_w, a, b, self.A_log,
                self.dt_bias, self.state, o, o_bf16)
        if z is None:
            check("ix_gdn_prefill", ix_gdn_prefill(*args, self._ws, self._ws.numel(), stream))
        else:
            g = out_gate(z, self.ssm_norm, self.norm_eps, y, y_bf16, y_q8_1)
            check("ix_gdn_prefill_gated", ix_gdn_prefill_gated(*args, g, self._ws, self._ws.numel(), stream))


def _check_rows(t, T, n):
    """Raises unless t is on the GPU as rows [T] of n bf16 values or more, dense but for the stride between them."""
    if t.dim() != 2 or t.stride(1) != 1 or t.dtype is not torch.bfloat16 or not t.is_cuda:
        _rows(t)
    if t.numel() < T * n or (T > 1 and t.stride(0) < n):
        raise ValueError("baloon_amd: rows are [heads][d], one behind the other")


class AttnLayer:
    """Attention of n_slots sequences of at most max_len tokens, h_q query heads over h_kv cached ones of d channels.

    Slot i has pages i * width .. of the cache to itself; with n_pages the caller keeps the pages instead and fills
    `table` [n_slots][width] int32 before they are needed. kv_len [n_slots] int32 counts the tokens held: setting it to 0
    empties a slot, to fewer tokens drops the last ones (rejected drafts). Tokens behind max_len are dropped.

    All of a call is on one stream, the lengths and a new o among it: `stream` (a torch stream or an address), or torch's
    current one. The caller orders calls on different streams, and what else it does with the layer's tensors. The workspace
    is allocated here for any batch (38 to 81 MiB), so a captured call's stays where it is."""

    def __init__(self, n_slots: int, max_len: int, h_q=16, h_kv=2, d=256, page=64, n_pages=None, window=0, sinks=0,
                 scale=None, device="cuda"):
        self.n_slots, self.h_q, self.h_kv, self.d = n_slots, h_q, h_kv, d
        self.window, self.sinks, self.scale = window, sinks, d ** -0.5 if scale is None else scale
        self.device = torch.device(device)
        self.width = -(-max_len // page)

        def tensor(*shape, dtype):
            return torch.zeros(*shape, dtype=dtype, device=self.device)

        pages = n_slots * self.width if n_pages is None else n_pages
        self.cache = kv8_cache(tensor(pages, h_kv, page, d, dtype=torch.int8), tensor(pages, h_kv, d, page, dtype=torch.int8),
                               tensor(pages, h_kv, dtype=torch.float32), tensor(pages, h_kv, dtype=torch.float32))
        self.table = tensor(n_slots, self.width, dtype=torch.int32)
        if n_pages is None:
            self.table.copy_(torch.arange(pages, dtype=torch.int32).view(n_slots, self.width))
        else:
            self.table.fill_(-1)
        self.kv_len = tensor(n_slots, dtype=torch.int32)
        self._one_each = torch.arange(n_slots + 1, dtype=torch.int32, device=self.device)
        most = min(2 ** 31 - 1, 2 ** 37 // max(h_q, 1))       # tokens of a call
        self._ws_bytes = ix_kv8_attn_workspace_size(self.cache, n_slots, most, most, h_q)
        self._ws = torch.empty(max(self._ws_bytes, 256), dtype=torch.uint8, device=self.device)

    def prefill(self, cu_seqlens, max_q, q, k, v, gate=None, o=None, stream=None):
        """Appends packed new tokens (cu_seqlens int32 [n_slots + 1] on the device, at most max_q of a sequence) and
        returns their attention o [T][h_q][d] bf16. q and gate are rows of [h_q][d], k and v of [h_kv][d], bf16, with any
        stride between rows; gate multiplies by its sigmoid."""
        if cu_seqlens.shape != (self.n_slots + 1,):
            raise ValueError("baloon_amd: cu_seqlens has an offset for each sequence and one more")
        if cu_seqlens.dtype != torch.int32 or not cu_seqlens.is_cuda or not cu_seqlens.is_contiguous():
            raise ValueError("baloon_amd: cu_seqlens is int32, contiguous and on the GPU")
        return self._on(stream, cu_seqlens, max_q, q, k, v, gate, o)

    def decode(self, q, k, v, gate=None, o=None, stream=None):
        """The same for one token of every sequence."""
        if q.shape[0] != self.n_slots:
            raise ValueError("baloon_amd: one token for each sequence")
        return self._on(stream, self._one_each, 1, q, k, v, gate, o)

    def _on(self, stream, *args):
        if stream is None:
            return self._attend(*args)
        if not isinstance(stream, torch.cuda.Stream):
            address = getattr(stream, "cuda_stream", getattr(stream, "value", stream)) or 0      # also a ctypes.c_void_p
            # torch takes an ExternalStream of address 0 for one that it is to choose
            stream = torch.cuda.ExternalStream(address, self.device) if address else torch.cuda.default_stream(self.device)
        with torch.cuda.stream(stream):
            return self._attend(*args)

    def _attend(self, cu_seqlens, max_q, q, k, v, gate, o):
        # What the calls below would refuse, or read and write beside the operands, is refused before anything is done.
        T = q.shape[0]
        if k.shape[0] != T or v.shape[0] != T or (gate is not None and gate.shape[0] != T):
            raise ValueError("baloon_amd: q, k, v and gate have a row for each token")
        for t, heads in ((q, self.h_q), (k, self.h_kv), (v, self.h_kv), (gate, self.h_q)):
            if t is not None:
                _check_rows(t, T, heads * self.d)
        if o is None:
            o = torch.empty(T, self.h_q, self.d, dtype=torch.bfloat16, device=self.device)
        elif o.dtype != torch.bfloat16 or not o.is_cuda or not o.is_contiguous() or o.numel() < T * self.h_q * self.d:
            raise ValueError("baloon_amd: o is bf16 [T][h_q][d], contiguous and on the GPU")
        if not self._ws_bytes or max_q < min(T, 1) or max_q >= 2 ** 31:
            check("ix_kv8_attn", HIP_ERROR_INVALID_VALUE)
        new = 1 if cu_seqlens is self._one_each else cu_seqlens.diff()
        where = (cu_seqlens, self.kv_len, self.table, self.width)
        self.kv_len += new
        try:
            check("ix_kv8_append", ix_kv8_append(self.cache, self.n_slots, T, *where, k, v))
            check("ix_kv8_attn", ix_kv8_attn(self.cache, self.n_slots, T, max_q, *where, q, self.h_q, self.scale, self.window,
                                             self.sinks, gate, o, self._ws, self._ws.numel()))
        except BaseException:
            self.kv_len -= new                                # a call that raises leaves the lengths as they were
            raise
        return o
