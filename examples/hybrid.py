"""A small hybrid stack, one attention layer to every three GDN layers, from prompts to generated tokens.

Between the layers the residual sum and the norm of the next one's input are one launch (ix_add_rms_norm). The attention
layer keeps its keys and values in the 8-bit cache (AttnLayer) and its output is gated, the GDN layers their states
(GdnLayer). Projections of prompts are torch products, those of single tokens ix_gdn_in_proj and ix_mmvq_q8_0, which
reads the last norm's q8_1 output. With rope_base the attention's queries and keys are normed and turned by position, and
several continuations of a prompt may go on from one pass over it. Weights are random: run it with
``python -m examples.hybrid``.
"""
import torch
import torch.nn.functional as F

import baloon_amd as bx


class Hybrid:
    def __init__(self, n_slots, max_len, hidden=1024, n_layers=4, h_q=8, h_kv=2, d=128, vocab=512, seed=0, rope_base=None,
                 **attention):
        self.n, self.hidden, self.h_q, self.h_kv, self.d, self.vocab = n_slots, hidden, h_q, h_kv, d, vocab
        self.cfg = c = bx.make_cfg(h_k=4, h_v=8)
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(rows, cols):
            return (torch.randn(rows, cols, generator=g, device="cuda") * cols ** -0.5).bfloat16()

        if rope_base:
            freq = bx.rope_freq(d // 2, rope_base)[0].cuda()                             # half of the channels turn
            q_norm, k_norm = (torch.randn(d, generator=g, device="cuda") * 0.1 for _ in "qk")
            attention.update(rope=bx.rope(freq, norm=q_norm, norm_offset=1.0), rope_k=bx.rope(freq, norm=k_norm, norm_offset=1.0))
        self.embed = weight(vocab, hidden) * hidden ** 0.5
        self.layers, last = [], None
        for i in range(n_layers):
            norm = (torch.randn(hidden, generator=g, device="cuda") * 0.1)               # its weight is 1 + norm
            if i % 4 == 3:
                w_in = weight((2 * h_q + 2 * h_kv) * d, hidden)                          # q | gate | k | v
                last = bx.AttnLayer(n_slots, max_len, h_q, h_kv, d, beside=last, **attention)       # the stack's layers run one after the other
                self.layers.append((last, norm, w_in, weight(hidden, h_q * d)))
            else:
                layer = bx.GdnLayer(n_slots, c)
                layer.conv_w.copy_(weight(c.channels, c.d_conv))
                layer.A_log.normal_(generator=g)
                layer.dt_bias.normal_(generator=g)
                w_in = weight(bx.ix_gdn_in_proj_width(c), hidden)                        # x | z | a | b
                self.layers.append((layer, norm, w_in, weight(hidden, c.h_v * c.d_v)))
        self.last_norm = torch.zeros(hidden, device="cuda")
        # the output matrix in Q8_0: per 32 weights an fp16 scale and 32 codes
        w = weight(vocab, hidden).float().view(vocab, hidden // 32, 32)
        scale = w.abs().amax(2, keepdim=True) / 127
        codes = torch.round(w / scale).to(torch.int8)
        self.head = torch.cat([scale.half().view(torch.uint8), codes.view(torch.uint8)], 2).contiguous()

    def norm(self, x, res, weight, y=None, y_q8_1=None):
        """(x + res, its norm), in one launch; x the last layer's output, or None before the first."""
        total = torch.empty_like(res)
        x, res = (res, None) if x is None else (x, res)
        bx.check("ix_add_rms_norm", bx.ix_add_rms_norm(total.shape[0], self.hidden, x, res, total, weight, 1.0, 1e-6, None, y, y_q8_1))
        return total

    def forward(self, tokens, cu=None, max_q=1):
        """Packed new tokens (or one for each sequence, cu None) to the logits of every sequence's last one."""
        T, c = tokens.shape[0], self.cfg
        res, out = self.embed[tokens], None
        for layer, weight, w_in, w_out in self.layers:
            h = torch.empty(T, self.hidden, dtype=torch.bfloat16, device="cuda")
            res = self.norm(out, res, weight, y=h)
            if isinstance(layer, bx.AttnLayer):
                qw, kw = self.h_q * self.d, self.h_kv * self.d
                q, gate, k, v = F.linear(h, w_in).split([qw, qw, kw, kw], 1)             # rows of one wide tensor
                y = layer.decode(q, k, v, gate) if cu is None else layer.prefill(cu, max_q, q, k, v, gate)
            else:
                Z = c.h_v * c.d_v
                y = torch.empty(T, Z, dtype=torch.bfloat16, device="cuda")
                if cu is None:
                    x, z = (torch.empty(T, n, dtype=torch.bfloat16, device="cuda") for n in (c.channels, Z))
                    a, b = (torch.empty(T, c.h_v, dtype=torch.bfloat16, device="cuda") for _ in "ab")
                    bx.check("ix_gdn_in_proj", bx.ix_gdn_in_proj(c, T, self.hidden, h, w_in, x, z, a, b))
                    layer.decode(x, a, b, z=z, y_bf16=y)
                else:
                    x, z, a, b = (t.contiguous() for t in F.linear(h, w_in).split([c.channels, Z, c.h_v, c.h_v], 1))
                    layer.prefill(cu, x, a, b, z=z, y_bf16=y)
            out = F.linear(y.view(T, -1), w_out)
        if cu is not None:
            at = (cu[1:] - 1).long()
            res, out = res[at], out[at]
        q8 = torch.empty(self.n * self.hidden // 32 * 36, dtype=torch.uint8, device="cuda")
        self.hidden_state = torch.empty_like(res)
        self.norm(out, res, self.last_norm, y=self.hidden_state, y_q8_1=q8)
        logits = torch.empty(self.n, self.vocab, dtype=torch.float32, device="cuda")
        bx.check("ix_mmvq_q8_0", bx.ix_mmvq_q8_0(self.head, q8, logits, self.hidden, self.vocab, self.n))
        return logits


    def fork(self, slot, n, tokens):
        """Slots slot .. slot + n - 1 go on from the `tokens` tokens that `slot` holds, all of them."""
        for layer, *_ in self.layers:
            if isinstance(layer, bx.AttnLayer):
                layer.fork(slot, n, tokens)
            else:
                for t in (layer.state, layer.conv_state):
                    t[slot + 1:slot + n] = t[slot].clone()


def generate(prompts, steps, seed=0):
    """Greedy continuations of token lists, and the model."""
    lens = [len(p) for p in prompts]
    model = Hybrid(len(prompts), max(lens) + steps, seed=seed)
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    logits = model.forward(torch.tensor(sum(prompts, []), device="cuda"), cu, max(lens))
    made = []
    for _ in range(steps):
        made.append(logits.argmax(1))
        logits = model.forward(made[-1])
    return torch.stack(made, 1).tolist(), model


def continuations(prompts, each, steps, seed=0, **attention):
    """`each` continuations of every prompt from one pass over it, drawn by the last token's logits, and the model (whose attention
    layers take what else is given)."""
    lens, n = [len(p) for p in prompts], len(prompts) * each
    model = Hybrid(n, max(lens) + steps, seed=seed, rope_base=1e4, max_forks=len(prompts), **attention)
    cu = torch.tensor([0] + [x for m in lens for x in (m, *[0] * (each - 1))], dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    logits = model.forward(torch.tensor(sum(prompts, []), device="cuda"), cu, max(lens))     # a slot without tokens: of those before it
    for i, m in enumerate(lens):
        if each > 1:
            model.fork(i * each, each, m)
    g, made = torch.Generator(device="cuda").manual_seed(seed), []
    for _ in range(steps):
        made.append(torch.multinomial(logits.softmax(1), 1, generator=g)[:, 0])
        logits = model.forward(made[-1])
    return torch.stack(made, 1).tolist(), model


if __name__ == "__main__":
    tokens, _ = generate([[i % 512 for i in range(5, 305)], [1, 2, 3], list(range(64))], 16)
    for t in tokens:
        print(*t)
    tokens, _ = continuations([[i % 512 for i in range(5, 305)], [1, 2, 3]], 3, 16)
    for t in tokens:
        print(*t)
