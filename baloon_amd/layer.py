"""GdnLayer and AttnLayer: device-resident parameters and per-sequence states of one layer.

GdnLayer is a thin host object over the C ABI: it owns the conv weights, A_log, dt_bias, the recurrent
state block [n][h_v][d_v][d_k] fp32 (each head's state stored column by column), the conv
state [n][C][d_conv-1] bf16, the gated output norm's weight ssm_norm [d_v] fp32 and the
zeroed decode workspace, and calls ``ix_gdn_decode`` / ``ix_gdn_prefill`` (or their gated
variants, when a gate input z is passed) on the current stream. Allocation happens here, at
construction (and for the prefill workspace, on first use of a given size), never inside the
library calls.

AttnLayer is the same for the softmax attention layers that stand between GDN layers: it owns a paged 8-bit
cache of keys and values and the lengths of its sequences, and calls ``ix_kv8_append`` and ``ix_kv8_attn``; with rotary
positions ``ix_kv8_append_rope``, and for sequences that were forked from one prompt ``ix_kv8_attn_shared``.
"""
from __future__ import annotations

import torch

from . import (HIP_ERROR_INVALID_VALUE, Cfg, _rows, check, ix_gdn_decode, ix_gdn_decode_gated, ix_gdn_decode_workspace_size, ix_gdn_prefill,
               ix_gdn_prefill_gated, ix_gdn_prefill_gated_workspace_size, ix_gdn_prefill_workspace_size,
               ix_kv8_append, ix_kv8_append_rope, ix_kv8_attn, ix_kv8_attn_shared, ix_kv8_attn_shared_workspace_size,
               ix_kv8_attn_workspace_size, kv8_cache, make_cfg, out_gate)


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
    is allocated here for any batch (38 to 81 MiB), so a captured call's stays where it is. Layers whose calls are ordered, as those
    of a stack are, need one between them: `beside`, another layer, whose workspaces this one takes where they are large enough.

    rope (``baloon_amd.rope``) norms and turns queries by position before they attend, rope_k (rope itself if not given) keys
    before they are stored. With max_forks, up to so many groups of slots may share a prompt (`fork`), which calls of up to 16
    new tokens a slot in the mean then read once for all of them, where that is worth it (`worth`: codes of keys that need
    not be read again), with a workspace of their own (57, 202 and 420 MiB for 4, 64 and 256 slots of 2 heads of 256)."""

    def __init__(self, n_slots: int, max_len: int, h_q=16, h_kv=2, d=256, page=64, n_pages=None, window=0, sinks=0,
                 scale=None, device="cuda", rope=None, rope_k=None, max_forks=0, worth=200_000_000, beside=None):
        self.n_slots, self.h_q, self.h_kv, self.d = n_slots, h_q, h_kv, d
        self.window, self.sinks, self.scale = window, sinks, d ** -0.5 if scale is None else scale
        self.device = torch.device(device)
        self.width = -(-max_len // page)
        self._own_pages = n_pages is None

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
        if beside is not None and not isinstance(beside, AttnLayer):
            raise ValueError("baloon_amd: beside is another AttnLayer")

        def workspace(n, theirs):
            if theirs is not None and theirs.numel() >= n and theirs.device == self.kv_len.device:
                return theirs
            return torch.empty(max(n, 256), dtype=torch.uint8, device=self.device)

        self._ws = workspace(self._ws_bytes, getattr(beside, "_ws", None))
        if rope is None and rope_k is not None:
            raise ValueError("baloon_amd: rope_k goes with rope")
        self.rope, self.rope_k = rope, rope if rope_k is None else rope_k
        if max_forks < 0 or (max_forks and window):
            raise ValueError("baloon_amd: forked sequences see all of their prompt: no window")
        self.max_forks, self.worth, self._forks, self._n_groups, self._shared_pays = max_forks, worth, {}, 0, False
        if max_forks:
            most = 2 * max_forks                              # groups: the forks, and what lies between two
            self._groups, self._shared = tensor(most + 1, dtype=torch.int32), tensor(most, dtype=torch.int32)
            self._few = 16 * n_slots
            n = ix_kv8_attn_shared_workspace_size(self.cache, n_slots, self._few, self._few, most, h_q)
            self._shared_ws = workspace(n, getattr(beside, "_shared_ws", None))

    def fork(self, slot, n, tokens, stream=None):
        """Slots slot + 1 .. slot + n - 1 go on from the first `tokens` tokens of `slot`, which holds as many, and from nothing that
        they held: its whole pages are theirs too, the page that the tokens end in is copied. Until `release`, none of the n may lose one of these
        tokens (a shorter kv_len, then new tokens). Not to be captured; calls that were captured before stay right, but take
        no more groups together than there were: with more forks, or where sharing has come to pay, capture them again."""
        others = range(slot + 1, slot + n)
        if slot < 0 or n < 2 or slot + n > self.n_slots or not 0 < tokens <= self.width * self.cache.page:
            raise ValueError("baloon_amd: a fork is of two slots or more, and of tokens that a slot can hold")
        if len(self._forks) >= self.max_forks:
            raise ValueError("baloon_amd: more than max_forks forks")
        if any(slot < s + m and s < slot + n for s, (m, _) in self._forks.items()):
            raise ValueError("baloon_amd: a slot of a fork already")
        self._on(stream, self._fork, slot, others, tokens)

    def _fork(self, slot, others, tokens):
        whole, rest = divmod(tokens, self.cache.page)
        if int(self.kv_len[slot]) < tokens:
            raise ValueError("baloon_amd: the slot holds fewer tokens")
        if rest:
            source, *pages = self.table[slot:others.stop, whole].tolist()
            if not all(0 <= p < self.cache.n_pages for p in (source, *pages)) or source in pages or len(set(pages)) < len(pages):
                raise ValueError("baloon_amd: the page that the tokens end in has no place of its own in each slot")
            for t in self.cache.tensors:
                t[pages] = t[source].clone()
        self._forks[slot] = (len(others) + 1, tokens)
        self._regroup()
        self.table[slot + 1:others.stop, :whole] = self.table[slot, :whole].clone()
        self.kv_len[slot + 1:others.stop] = tokens

    def release(self, slot, stream=None):
        """Ends the fork of `slot`: the others of it are empty again, with pages of their own (where the caller keeps the
        pages, without those that they shared)."""
        if slot not in self._forks:
            raise ValueError("baloon_amd: not a slot that others were forked from")
        self._on(stream, self._release, slot)

    def _release(self, slot):
        n, tokens = self._forks.pop(slot)
        whole = tokens // self.cache.page
        rows = self.table[slot + 1:slot + n, :whole]
        if self._own_pages:
            first = torch.arange(slot + 1, slot + n, dtype=torch.int32, device=self.device)[:, None] * self.width
            rows.copy_(first + torch.arange(whole, dtype=torch.int32, device=self.device))
        else:
            rows.fill_(-1)
        self.kv_len[slot + 1:slot + n] = 0
        self._regroup()

    def _regroup(self):
        """The groups of ix_kv8_attn_shared lie side by side: between two forks is one that shares nothing."""
        ends, shared = [], []
        for slot, (n, tokens) in sorted(self._forks.items()):
            if ends and ends[-1] < slot:
                ends.append(slot)
                shared.append(0)
            ends += [slot + n] if ends else [slot, slot + n]
            shared.append(tokens)
        self._n_groups = len(shared)
        # Reading shared tokens once pays from about 2e8 codes of keys on that need not be read again (below that it may pay, too: 42 us
        # and 79 for 68 tokens in 17 groups behind 6,500; or not: 39 and 19 for 138 times 5 in 23 behind 90). us with and without, 37
        # sequences of 4 new tokens, 32 heads over 8 of 128, behind 4,096 tokens 48 and 44, behind 8,192 59 and 83; 64 of one,
        # 16 over 2 of 256, behind 2,048, 4,096 and 8,190 32, 42, 49 and 30, 41, 62; 24 times 4 behind 300 to 6,000 55 and 101.
        self._shared_pays = sum((n - 1) * tokens for n, tokens in self._forks.values()) * self.h_kv * self.d >= self.worth
        # A captured call has the groups that there were then: what is more than there are now is empty and shares nothing.
        ends += [ends[-1] if ends else 0] * (len(self._groups) - len(ends))
        self._groups.copy_(torch.tensor(ends, dtype=torch.int32))
        self._shared.copy_(torch.tensor(shared + [0] * (len(self._shared) - len(shared)), dtype=torch.int32))

    def prefill(self, cu_seqlens, max_q, q, k, v, gate=None, o=None, stream=None):
        """Appends packed new tokens (cu_seqlens int32 [n_slots + 1] on the device, at most max_q of a sequence) and
        returns their attention o [T][h_q][d] bf16. q and gate are rows of [h_q][d], k and v of [h_kv][d], bf16, with any
        stride between rows; gate multiplies by its sigmoid."""
        if cu_seqlens.shape != (self.n_slots + 1,):
            raise ValueError("baloon_amd: cu_seqlens has an offset for each sequence and one more")
        if cu_seqlens.dtype != torch.int32 or not cu_seqlens.is_cuda or not cu_seqlens.is_contiguous():
            raise ValueError("baloon_amd: cu_seqlens is int32, contiguous and on the GPU")
        return self._on(stream, self._attend, cu_seqlens, max_q, q, k, v, gate, o)

    def decode(self, q, k, v, gate=None, o=None, stream=None):
        """The same for one token of every sequence."""
        if q.shape[0] != self.n_slots:
            raise ValueError("baloon_amd: one token for each sequence")
        return self._on(stream, self._attend, self._one_each, 1, q, k, v, gate, o)

    def _on(self, stream, call, *args):
        if stream is None:
            return call(*args)
        if not isinstance(stream, torch.cuda.Stream):
            address = getattr(stream, "cuda_stream", getattr(stream, "value", stream)) or 0      # also a ctypes.c_void_p
            # torch takes an ExternalStream of address 0 for one that it is to choose
            stream = torch.cuda.ExternalStream(address, self.device) if address else torch.cuda.default_stream(self.device)
        with torch.cuda.stream(stream):
            return call(*args)

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
            if self.rope is None:
                check("ix_kv8_append", ix_kv8_append(self.cache, self.n_slots, T, *where, k, v))
            else:
                turned = torch.empty(T, self.h_q, self.d, dtype=torch.bfloat16, device=self.device)      # not o: that may be the gate's
                check("ix_kv8_append_rope", ix_kv8_append_rope(self.cache, self.n_slots, T, *where, k, v, self.rope_k, q, self.h_q,
                                                               self.rope, turned))
                q = turned
            if self._shared_pays and T <= self._few:
                check("ix_kv8_attn_shared", ix_kv8_attn_shared(self.cache, self.n_slots, T, min(max_q, T), *where, self._n_groups,
                                                               self._groups, self._shared, q, self.h_q, self.scale, gate, o,
                                                               self._shared_ws, self._shared_ws.numel()))
            else:
                check("ix_kv8_attn", ix_kv8_attn(self.cache, self.n_slots, T, max_q, *where, q, self.h_q, self.scale, self.window,
                                                 self.sinks, gate, o, self._ws, self._ws.numel()))
        except BaseException:
            self.kv_len -= new                                # a call that raises leaves the lengths as they were
            raise
        return o
