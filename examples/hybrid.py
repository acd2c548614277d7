"""A small hybrid stack, one attention layer to every three GDN layers, from prompts to generated tokens.

Between the layers the residual sum and the norm of the next one's input are one launch (ix_add_rms_norm). The attention
layer keeps its keys and values in the 8-bit cache (AttnLayer) and its output is gated, the GDN layers their states
(GdnLayer). Projections of prompts are torch products, those of single tokens ix_gdn_in_proj and ix_mmvq_q8_0, which
reads the last norm's q8_1 output. Weights are random: run it with ``python -m examples.hybrid``.
"""
import torch
import torch.nn.functional as F

import baloon_amd as bx


class Hybrid:
    def __init__(self, n_slots, max_len, hidden=1024, n_layers=4, h_q=8, h_kv=2, d=128, vocab=512, seed=0):
        self.n, self.hidden, self.h_q, self.h_kv, self.d, self.vocab = n_slots, hidden, h_q, h_kv, d, vocab
        self.cfg = c = bx.make_cfg(h_k=4, h_v=8)
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(rows, cols):
            return (torch.randn(rows, cols, generator=g, device="cuda") * cols ** -0.5).bfloat16()

        self.embed = weight(vocab, hidden) * hidden ** 0.5
        self.layers = []
        for i in range(n_layers):
            norm = (torch.randn(hidden, generator=g, device="cuda") * 0.1)               # its weight is 1 + norm
            if i % 4 == 3:
                w_in = weight((2 * h_q + 2 * h_kv) * d, hidden)                          # q | gate | k | v
                self.layers.append((bx.AttnLayer(n_slots, max_len, h_q, h_kv, d), norm, w_in, weight(hidden, h_q * d)))
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


if __name__ == "__main__":
    tokens, _ = generate([[i % 512 for i in range(5, 305)], [1, 2, 3], list(range(64))], 16)
    for t in tokens:
        print(*t)
