"""Performance cases of the operators that stand between the GDN layers of a hybrid model: the residual
addition with its RMS norm, the key/value cache in 8 bits, and the attention that reads it.

    own                 False: run() computes the plain form in elementary torch operations, in 32 bits;
                        True: run() calls the library
    listed()            the named cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) the inputs, cache and workspaces a program holds before the call
    run(state)          one pass; returns every output
    work(case)          bytes and operations that one pass cannot do without
    exact(case, seed)   run's results in 64-bit arithmetic

A case is a dict of plain values. "kind" picks the operator:

    norm    h = x + residual, y = RMS norm of h, as bf16 or as q8_1 blocks (32 codes with an fp16 scale)
    append  keys and values of new tokens into the paged 8-bit cache, and the pages read back
    attn    attention of new tokens over the cached ones: single tokens, drafted windows, prompts

The cache holds pages of `page` tokens: codes k [n_pages][h_kv][page][d] and v [n_pages][h_kv][d][page]
(int8), scales [n_pages][h_kv] (fp32, one per page and head). table [n_seq][width] names a sequence's pages.
A sequence of kv_len tokens whose last q_len are the new ones: query i stands at position
kv_len - q_len + i.
"""
import math
import random

import torch

own = False

EPS = 1e-6


# ---------------------------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------------------------
# Lengths of a batch: q_lo..q_hi new tokens and c_lo..c_hi cached ones before them, drawn evenly from
# lens_seed. Head layouts: 16 query and 2 key/value heads of 256, the attention layers that go with the
# 2,048-wide GDN model of 16 and 32 heads; others are tensor-parallel shares and common ones.

def listed():
    return [
        # A single user's token: the norm ahead of a layer, 2,048 wide. Latency.
        dict(name="norm_1", kind="norm", rows=1, n=2048, x="bf16", y="bf16"),
        # A quantised model's small batch: the fp32 result of a Q8_0 product is added, and the norm leaves
        # in q8_1 for the next product.
        dict(name="norm_q8_8", kind="norm", rows=8, n=4096, x="f32", y="q8_1"),
        # The residual stream of a prompt.
        dict(name="norm_8192", kind="norm", rows=8192, n=2048, x="bf16", y="bf16"),
        # One new token for each of 64 sequences: the page's scale grows or stays, its codes follow.
        dict(name="append_64", kind="append", n_seq=64, q_lo=1, q_hi=1, c_lo=1, c_hi=4096, lens_seed=1, h_kv=2, d=256,
             page=16),
        # Prompts of a prefill batch into fresh and half-filled pages.
        dict(name="append_varlen_16", kind="append", n_seq=16, q_lo=1, q_hi=2048, c_lo=0, c_hi=100, lens_seed=2,
             h_kv=2, d=256, page=64),
        # A single user's token after a thousand others. Latency.
        dict(name="attn_1", kind="attn", n_seq=1, q_lo=1, q_hi=1, c_lo=1000, c_hi=1000, lens_seed=3, h_q=16, h_kv=2,
             d=256, page=16, window=0, sinks=0, gate=True),
        # The serving batch: 64 sequences of all lengths, one token each.
        dict(name="attn_64", kind="attn", n_seq=64, q_lo=1, q_hi=1, c_lo=1, c_hi=8192, lens_seed=4, h_q=16, h_kv=2,
             d=256, page=16, window=0, sinks=0, gate=True),
        # One token at the end of a long document.
        dict(name="attn_long", kind="attn", n_seq=1, q_lo=1, q_hi=1, c_lo=262143, c_hi=262143, lens_seed=5, h_q=16,
             h_kv=2, d=256, page=64, window=0, sinks=0, gate=False),
        # Speculative decoding: four drafted tokens for each of 37 sequences.
        dict(name="attn_window_37x4", kind="attn", n_seq=37, q_lo=4, q_hi=4, c_lo=100, c_hi=4000, lens_seed=6, h_q=32,
             h_kv=8, d=128, page=32, window=0, sinks=0, gate=False),
        # Layers that see the last 1,024 tokens and the first four, in a batch of long sequences.
        dict(name="attn_sinks_48", kind="attn", n_seq=48, q_lo=1, q_hi=1, c_lo=500, c_hi=12000, lens_seed=7, h_q=20,
             h_kv=4, d=128, page=16, window=1024, sinks=4, gate=False),
        # One prompt of 4,096 tokens.
        dict(name="attn_prompt_4096", kind="attn", n_seq=1, q_lo=4096, q_hi=4096, c_lo=0, c_hi=0, lens_seed=8, h_q=16,
             h_kv=2, d=256, page=16, window=0, sinks=0, gate=True),
        # A batch of prompt pieces behind cached ones.
        dict(name="attn_varlen_8", kind="attn", n_seq=8, q_lo=1, q_hi=1500, c_lo=0, c_hi=3000, lens_seed=9, h_q=16,
             h_kv=4, d=128, page=64, window=0, sinks=0, gate=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    case = _drawn(rng)
    while case["kind"] == "attn" and (work(case)["flops"] > 1.3e11 or work(case)["bytes"] > 2.6e8):   # of the largest listed
        case.update(q_hi=-(-2 * case["q_hi"] // 3), q_lo=-(-2 * case["q_lo"] // 3), c_hi=-(-2 * case["c_hi"] // 3))
        case["c_lo"] = min(case["c_lo"], case["c_hi"])
    return case


def _drawn(rng):
    kind = rng.choice(["norm", "append", "attn", "attn", "attn", "attn"])
    if kind == "norm":
        if rng.random() < 0.35:
            return dict(kind=kind, rows=rng.randint(1, 8), n=32 * _log_int(rng, 16, 256), x=rng.choice(["f32", "bf16"]),
                        y="q8_1")
        n = _log_int(rng, 500, 8192)
        return dict(kind=kind, rows=_log_int(rng, 1, 2 ** 24 // n), n=n, x=rng.choice(["bf16", "bf16", "f32"]), y="bf16")
    heads, d = rng.choice([(2, 256), (2, 256), (1, 256), (8, 128), (4, 128), (2, 128), (8, 64)])
    page, lens_seed = rng.choice([16, 16, 32, 64]), rng.randrange(1 << 16)
    if kind == "append":
        if rng.random() < 0.5:
            q = rng.choice([1, 1, 1, rng.randint(2, 8)])
            return dict(kind=kind, n_seq=_log_int(rng, 1, 256), q_lo=q, q_hi=q, c_lo=0, c_hi=_log_int(rng, 16, 8192),
                        lens_seed=lens_seed, h_kv=heads, d=d, page=page)
        return dict(kind=kind, n_seq=rng.randint(1, 16), q_lo=1, q_hi=_log_int(rng, 10, 2048), c_lo=0, c_hi=100,
                    lens_seed=lens_seed, h_kv=heads, d=d, page=page)
    group = rng.choice([8, 8, 4, 4, 5, 1, 16]) if d == 256 else rng.choice([4, 4, 8, 5, 1])
    window, sinks = rng.choice([(0, 0), (0, 0), (0, 0), (_log_int(rng, 100, 4096), rng.choice([0, 1, 4, 17]))])
    more = dict(lens_seed=lens_seed, h_q=group * heads, h_kv=heads, d=d, page=page, window=window, sinks=sinks,
                gate=rng.random() < 0.5)
    what = rng.choice(["token", "token", "drafts", "prompts", "long"])
    if what == "long":
        c = _log_int(rng, 8192, 131072)
        return dict(kind=kind, n_seq=1, q_lo=1, q_hi=1, c_lo=c, c_hi=c, **more)
    if what == "prompts":
        n_seq = rng.choice([1, 1, rng.randint(2, 8)])
        q = _log_int(rng, 20, 2500 if n_seq == 1 else 1000)
        return dict(kind=kind, n_seq=n_seq, q_lo=q if n_seq == 1 else 1, q_hi=q, c_lo=0,
                    c_hi=rng.choice([0, rng.randint(1, 2000)]), **more)
    q = 1 if what == "token" else rng.randint(2, 8)
    return dict(kind=kind, n_seq=_log_int(rng, 1, 96), q_lo=q, q_hi=q, c_lo=1, c_hi=_log_int(rng, 16, 8192), **more)


def _lens(case):
    """(new tokens, tokens in all) of each sequence."""
    r = random.Random(case["lens_seed"])
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["n_seq"])]
    return q, [r.randint(case["c_lo"], case["c_hi"]) + n for n in q]


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------

class _Gen:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=self.g)

    def codes(self, *shape):
        """int8 codes as a quantiser leaves normal values: the largest of a block near 127."""
        t = torch.empty(*shape, dtype=torch.int8, device="cuda")
        t.view(-1).random_(-60, 61, generator=self.g)
        return t

    def scales(self, *shape):
        return torch.empty(*shape, device="cuda").uniform_(0.015, 0.04, generator=self.g)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cumulative(v):
    return [sum(v[:i]) for i in range(len(v) + 1)]


def _cache(case, g, kv):
    """The cache with every page's codes and scales filled, and a table of pages in no order."""
    page, h, d = case["page"], case["h_kv"], case["d"]
    pages = [-(-n // page) for n in kv]
    width, n_pages = max(pages) + 1, sum(pages) + 7
    order = g.order(n_pages)[:sum(pages)].to(torch.int32)
    table = torch.full((len(kv), width), -1, dtype=torch.int32, device="cuda")
    for b, at in enumerate(_cumulative(pages)[:-1]):
        table[b, :pages[b]] = order[at:at + pages[b]]
    return dict(k=g.codes(n_pages, h, page, d), v=g.codes(n_pages, h, d, page), k_scale=g.scales(n_pages, h),
                v_scale=g.scales(n_pages, h), table=table, width=width)


def prepare(case, seed):
    g = _Gen(seed)
    s = dict(case=case)
    if case["kind"] == "norm":
        rows, n = case["rows"], case["n"]
        s.update(x=g.normal(rows, n, dtype=torch.float32 if case["x"] == "f32" else torch.bfloat16), res=g.normal(rows, n, std=2.0),
                 w=g.normal(n, std=0.2, dtype=torch.float32), res_out=torch.empty(rows, n, dtype=torch.bfloat16, device="cuda"))
        if case["y"] == "q8_1":
            s["y"] = torch.empty(rows, n // 32, 36, dtype=torch.uint8, device="cuda")
        else:
            s["y"] = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
        return s
    q, kv = _lens(case)
    d, h, page = case["d"], case["h_kv"], case["page"]
    T = sum(q)
    s.update(_cache(case, g, kv), q_len=_ints(q), cu=_ints(_cumulative(q)), kv_len=_ints(kv), T=T)
    if case["kind"] == "append":
        # Keys and values as slices of one projection's rows, as a fused projection leaves them. Some
        # tokens are larger than what their page holds.
        rows = g.normal(T, 2 * h * d) * (1 + g.normal(T, 1, std=0.3).abs())
        s.update(new_k=rows[:, :h * d].view(T, h, d), new_v=rows[:, h * d:].view(T, h, d))
        # Pages are read back from the start of the first one that changes.
        back = [n - (n - m) // page * page for m, n in zip(q, kv)]
        s.update(back=_ints(back), back_cu=_ints(_cumulative(back)), back_T=sum(back),
                 out_k=torch.empty(sum(back), h, d, dtype=torch.bfloat16, device="cuda"),
                 out_v=torch.empty(sum(back), h, d, dtype=torch.bfloat16, device="cuda"))
    else:
        s.update(q=g.normal(T, case["h_q"], d, std=2.0), o=torch.empty(T, case["h_q"], d, dtype=torch.bfloat16, device="cuda"),
                 gate=g.normal(T, case["h_q"], d) if case["gate"] else None, max_q=max(q), max_kv=max(kv), scale=d ** -0.5)
    if own:                                      # the description and workspace that a program keeps beside its cache
        import baloon_amd as bx
        s["cache"] = bx.kv8_cache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if case["kind"] == "attn":
            n = bx.ix_kv8_attn_workspace_size(s["cache"], case["n_seq"], T, s["max_q"], case["h_q"])
            s["ws"] = torch.zeros(max(n, 1), dtype=torch.uint8, device="cuda")
    return s


# ---------------------------------------------------------------------------------------------
# The library's calls
# ---------------------------------------------------------------------------------------------

def _run_own(s):
    import baloon_amd as bx
    c = s["case"]
    if c["kind"] == "norm":
        y = {"y_q8_1" if c["y"] == "q8_1" else "y_bf16": s["y"]}
        bx.check("ix_add_rms_norm", bx.ix_add_rms_norm(c["rows"], c["n"], s["x"], s["res"], s["res_out"], s["w"], 1.0, EPS, **y))
        if c["y"] == "bf16":
            return dict(res=s["res_out"], y=s["y"])
        # the values that the codes stand for: scale times code
        return dict(res=s["res_out"], y=s["y"].view(torch.int8)[..., 4:] * s["y"].view(torch.float16)[..., :1])
    if c["kind"] == "append":
        bx.check("ix_kv8_append", bx.ix_kv8_append(s["cache"], c["n_seq"], s["T"], s["cu"], s["kv_len"], s["table"],
                                                   s["width"], s["new_k"], s["new_v"]))
        bx.check("ix_kv8_read", bx.ix_kv8_read(s["cache"], c["n_seq"], s["back_T"], s["back_cu"], s["kv_len"], s["table"],
                                               s["width"], s["out_k"], s["out_v"]))
        return dict(k=s["out_k"], v=s["out_v"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    bx.check("ix_kv8_attn", bx.ix_kv8_attn(s["cache"], c["n_seq"], s["T"], s["max_q"], s["cu"], s["kv_len"], s["table"],
                                           s["width"], s["q"], c["h_q"], s["scale"], c["window"], c["sinks"], s["gate"],
                                           s["o"], s["ws"], s["ws"].numel()))
    return dict(o=s["o"])


# ---------------------------------------------------------------------------------------------
# The plain form
# ---------------------------------------------------------------------------------------------

def _plain_norm(s):
    c = s["case"]
    h = (s["x"].float() + s["res"].float()).to(torch.bfloat16)
    f = h.float()
    y = f * (1.0 / torch.sqrt((f * f).mean(1, keepdim=True) + EPS)) * (s["w"] + 1.0)
    if c["y"] == "bf16":
        return dict(res=h, y=y.to(torch.bfloat16))
    y = y.view(c["rows"], -1, 32)
    d = y.abs().amax(2, keepdim=True) / 127.0
    codes = torch.where(d > 0, torch.floor(y.abs() / d + 0.5) * torch.sign(y), 0.0)
    return dict(res=h, y=(codes * d.half().float()).half())


def _tokens(lens, cu, T):
    """(sequence, place in it) of each of T packed rows."""
    b = torch.repeat_interleave(torch.arange(lens.numel(), device="cuda"), lens.long(), output_size=T)
    return b, torch.arange(T, device="cuda") - cu.long()[b]


def _plain_append(s):
    c, page = s["case"], s["case"]["page"]
    table, kv = s["table"].long(), s["kv_len"].long()
    b, i = _tokens(s["q_len"], s["cu"], s["T"])
    pos = (kv - s["q_len"])[b] + i
    at, slot = table[b, pos // page], pos % page
    # the first page of each sequence may hold older tokens, in its first `held` slots
    first = kv - s["q_len"]
    p0, held = table.gather(1, (first // page)[:, None])[:, 0], first % page
    older = torch.arange(page, device="cuda")[None, :] < held[:, None]
    s_k, s_v = s["k_scale"], s["v_scale"]

    def grow(x, scale):
        """The new scale of every page, and the old ones over the new for the first pages."""
        new = torch.zeros_like(scale)
        new.scatter_reduce_(0, at[:, None].expand(-1, x.shape[1]), x.float().abs().amax(2) / 127.0, "amax")
        old = torch.where(held[:, None] > 0, scale[p0], 0.0)
        touched = torch.zeros(scale.shape[0], dtype=torch.bool, device="cuda").index_fill_(0, at, True)
        new[p0] = torch.maximum(new[p0], old)
        new = torch.where(touched[:, None], new, scale)
        up = new[p0]
        return new, torch.where(up > old, old / up, 1.0)

    def codes(x, scale):
        d = scale[at][:, :, None]
        return torch.where(d > 0, torch.round(x.float() / d), 0.0).clamp(-127, 127).to(torch.int8)

    new_k, r_k = grow(s["new_k"], s_k)
    new_v, r_v = grow(s["new_v"], s_v)
    old_k, old_v = s["k"][p0], s["v"][p0]
    s["k"][p0] = torch.where(older[:, None, :, None], torch.round(old_k.float() * r_k[:, :, None, None]).to(torch.int8), old_k)
    s["v"][p0] = torch.where(older[:, None, None, :], torch.round(old_v.float() * r_v[:, :, None, None]).to(torch.int8), old_v)
    heads = torch.arange(c["h_kv"], device="cuda")[None, :]
    s["k"][at[:, None], heads, slot[:, None]] = codes(s["new_k"], new_k)
    s["v"][at[:, None], heads, :, slot[:, None]] = codes(s["new_v"], new_v)
    s_k.copy_(new_k)
    s_v.copy_(new_v)
    # and back
    b, i = _tokens(s["back"], s["back_cu"], s["back_T"])
    pos = (kv - s["back"])[b] + i
    at, slot = table[b, pos // page][:, None], (pos % page)[:, None]
    k = s["k"][at, heads, slot].float() * s_k[at, heads][:, :, None]
    v = s["v"][at, heads, :, slot].float() * s_v[at, heads][:, :, None]
    return dict(k=k.to(torch.bfloat16), v=v.to(torch.bfloat16), k_scale=s_k, v_scale=s_v)


def _plain_attn(s):
    c = s["case"]
    B, h, d, page, mq, mkv = c["n_seq"], c["h_kv"], c["d"], c["page"], s["max_q"], s["max_kv"]
    G = c["h_q"] // h
    q_len, kv, cu = s["q_len"].long(), s["kv_len"].long(), s["cu"].long()
    np_ = -(-mkv // page)
    pages = s["table"][:, :np_].long().clamp(min=0)
    k = s["k"][pages].float() * s["k_scale"][pages][..., None, None]            # [B, np, h, page, d]
    v = s["v"][pages].float() * s["v_scale"][pages][..., None, None]            # [B, np, h, d, page]
    k = k.permute(0, 2, 4, 1, 3).reshape(B, h, d, np_ * page)
    v = v.permute(0, 2, 1, 4, 3).reshape(B, h, np_ * page, d)
    i = torch.arange(mq, device="cuda")
    row = (cu[:-1, None] + i[None, :]).clamp(max=s["T"] - 1)
    q = s["q"][row].float() * s["scale"]                                        # [B, mq, h_q, d]
    q = q.view(B, mq, h, G, d).permute(0, 2, 1, 3, 4).reshape(B, h, mq * G, d)
    pos = (kv - q_len)[:, None, None] + i[None, :, None]
    j = torch.arange(np_ * page, device="cuda")[None, None, :]
    seen = (j <= pos) & (j < kv[:, None, None])
    if c["window"]:
        seen = seen & ((pos - j < c["window"]) | (j < c["sinks"]))
    seen = seen.repeat_interleave(G, 1)[:, None]
    a = torch.where(seen, torch.matmul(q, k), float("-inf"))
    top = a.amax(3, keepdim=True)
    a = torch.exp(a - torch.where(torch.isfinite(top), top, 0.0))
    total = a.sum(3, keepdim=True)
    o = torch.matmul(a, v) / torch.where(total > 0, total, 1.0)
    o = o.view(B, h, mq, G, d).permute(0, 2, 1, 3, 4).reshape(B, mq, c["h_q"], d)
    b, i = _tokens(s["q_len"], s["cu"], s["T"])
    o = o[b, i]
    if s["gate"] is not None:
        o = o / (1.0 + torch.exp(-s["gate"].float()))
    return dict(o=o.to(torch.bfloat16))


def run(state):
    if own:
        return _run_own(state)
    return {"norm": _plain_norm, "append": _plain_append, "attn": _plain_attn}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------

def work(case):
    if case["kind"] == "norm":
        rows, n = case["rows"], case["n"]
        x, y = 4 if case["x"] == "f32" else 2, 36 / 32 if case["y"] == "q8_1" else 2
        return dict(bytes=rows * n * (x + 2 + 2 + y) + 4 * n, flops=6 * rows * n)
    q, kv = _lens(case)
    h, d, page = case["h_kv"], case["d"], case["page"]
    if case["kind"] == "append":
        back = sum(n - (n - m) // page * page for m, n in zip(q, kv))
        # rows in, codes out; codes in, rows back out
        return dict(bytes=2 * h * d * (3 * sum(q) + 3 * back), flops=2 * h * d * (4 * sum(q) + back))
    pairs = tokens = 0
    for m, n in zip(q, kv):
        w, sinks = case["window"] or n, case["sinks"] if case["window"] else 0
        for p in range(n - m, n):
            pairs += min(w, p + 1) + min(sinks, max(0, p + 1 - w))
        first = max(0, n - m + 1 - w)                   # of the first query's window
        tokens += n - first + min(sinks, first)
    rows = sum(q) * case["h_q"] * d
    return dict(bytes=2 * tokens * h * d + 2 * rows * (3 if case["gate"] else 2), flops=4 * pairs * case["h_q"] * d)


# ---------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["kind"] == "norm":
        h = (s["x"].to(f64) + s["res"].to(f64)).to(torch.bfloat16)       # the stream is held in bf16
        z = h.to(f64)
        y = z / torch.sqrt((z ** 2).sum(1, keepdim=True) / case["n"] + EPS) * (1.0 + s["w"].to(f64))
        if case["y"] == "q8_1":
            blocks = y.reshape(case["rows"], case["n"] // 32, 32)
            d = blocks.abs().max(2, keepdim=True).values / 127
            y = torch.trunc(blocks / d + 0.5 * torch.sign(blocks)) * d.to(torch.float16).to(f64)   # halves away from zero
        return dict(res=h.to(f64), y=y)
    q, kv = _lens(case)
    h, d, page = case["h_kv"], case["d"], case["page"]
    cu = _cumulative(q)
    table = s["table"].cpu().tolist()
    if case["kind"] == "append":
        out = {"k": [], "v": []}
        scale = {"k": s["k_scale"].to(f64), "v": s["v_scale"].to(f64)}
        for b in range(case["n_seq"]):
            first, row = kv[b] - q[b], cu[b]
            for p in range(first // page, -(-kv[b] // page)):
                at, lo, hi = table[b][p], max(first, p * page), min(kv[b], (p + 1) * page)
                held, new = lo - p * page, hi - lo
                for name in ("k", "v"):
                    x = s["new_" + name][row:row + new].to(f64).transpose(0, 1)             # [h, new, d]
                    codes = s[name][at].to(f64)
                    if name == "v":
                        codes = codes.transpose(1, 2)
                    codes = codes[:, :held]
                    was = scale[name][at] if held else torch.zeros(h, dtype=f64, device="cuda")
                    now = torch.maximum(was, x.abs().amax((1, 2)) / 127)
                    now = torch.where(now > was, now.float().to(f64), now)                  # scales are held in 32 bits
                    codes = torch.cat([torch.round(codes * (was / now)[:, None, None]), torch.round(x / now[:, None, None])], 1)
                    out[name].append((codes * now[:, None, None]).transpose(0, 1))
                    scale[name][at] = now
                row += new
        return dict(k=torch.cat(out["k"]), v=torch.cat(out["v"]), k_scale=scale["k"], v_scale=scale["v"])
    G = case["h_q"] // h
    o = torch.zeros(sum(q), case["h_q"], d, dtype=f64, device="cuda")
    for b in range(case["n_seq"]):
        pages = s["table"][b, :-(-kv[b] // page)].long()
        pos = torch.arange(kv[b] - q[b], kv[b], device="cuda")[:, None]
        j = torch.arange(kv[b], device="cuda")[None, :]
        hidden = j > pos
        if case["window"]:
            hidden |= (j <= pos - case["window"]) & (j >= case["sinks"])
        for head in range(case["h_q"]):
            e = head // G
            k = (s["k"][pages, e].to(f64) * s["k_scale"][pages, e].to(f64)[:, None, None]).reshape(-1, d)[:kv[b]]
            v = (s["v"][pages, e].to(f64) * s["v_scale"][pages, e].to(f64)[:, None, None]).transpose(1, 2).reshape(-1, d)[:kv[b]]
            x = s["q"][cu[b]:cu[b + 1], head].to(f64)
            a = (x @ k.T * s["scale"]).masked_fill(hidden, float("-inf"))
            o[cu[b]:cu[b + 1], head] = torch.softmax(a, 1) @ v
    if s["gate"] is not None:
        o = o * torch.sigmoid(s["gate"].to(f64))
    return dict(o=o)
