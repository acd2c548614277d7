"""Performance cases of what an attention layer of a hybrid model does around its 8-bit key/value cache: rotary
positions (with the head's norm ahead of them), the append that turns keys and queries on the way, and the attention of a
batch whose sequences have their first tokens in common.

    own                 False: run() computes the plain form in elementary torch operations, in 32 bits;
                        True: run() calls the library
    listed()            the named cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) the inputs, cache and workspaces a program holds before the call
    run(state)          one pass; returns every output
    work(case)          bytes and operations that one pass cannot do without
    exact(case, seed)   run's results in 64-bit arithmetic

A case is a dict of plain values. "kind" picks the operator:

    rope    rows of heads: RMS norm of each head (if wanted), then its first `rot` channels turned by position
    append  the same on new keys and queries, keys and values into the paged 8-bit cache, and the pages read back
    shared  attention of new tokens over the cached ones; the sequences of a group have their first tokens in common

The cache holds pages of `page` tokens: codes k [n_pages][h_kv][page][d] and v [n_pages][h_kv][d][page]
(int8), scales [n_pages][h_kv] (fp32, one per page and head). table [n_seq][width] names a sequence's pages.
A sequence of kv_len tokens whose last q_len are the new ones: query i stands at position kv_len - q_len + i.
Channels turn in pairs by position * freq[i]: "halves" pairs channel i with i + rot / 2, "pairs" 2 i with 2 i + 1.
"""
import math
import random

import torch

own = False

EPS = 1e-6


# ---------------------------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------------------------
# Lengths of a batch: q_lo..q_hi new tokens and c_lo..c_hi cached ones before them, drawn evenly from lens_seed; for "shared" the
# cached ones come behind the s_lo..s_hi tokens of the sequence's group (groups of n_seq / n_groups sequences each).
# Head layouts: 16 query and 2 key/value heads of 256 with 64 channels turned and a norm for each head, the attention
# layers that go with the 2,048-wide GDN model; others are common ones.
# "scaling" is how the frequencies are made fit for contexts of `factor` times the length trained on: "none", "linear"
# (all divided), "parts" (long waves divided, short ones kept, those between in proportion; cosine and sine a little larger).

def listed():
    return [
        # A single user's token: the queries of one layer. Latency.
        dict(name="rope_1", kind="rope", n_seq=1, q_lo=1, q_hi=1, c_lo=1000, c_hi=1000, lens_seed=1, heads=16, d=256, rot=64,
             layout="halves", scaling="none", base=1e7, factor=1, norm=True, wide=20),
        # A prompt's queries, whole heads turned pair by pair.
        dict(name="rope_prompt_4096", kind="rope", n_seq=1, q_lo=4096, q_hi=4096, c_lo=0, c_hi=0, lens_seed=2, heads=32, d=128, rot=128,
             layout="pairs", scaling="none", base=1e4, factor=1, norm=False, wide=48),
        # Pieces of very long documents, frequencies scaled for them.
        dict(name="rope_far_6", kind="rope", n_seq=6, q_lo=1, q_hi=700, c_lo=200000, c_hi=1000000, lens_seed=3, heads=16, d=256, rot=64,
             layout="halves", scaling="parts", base=1e7, factor=4, norm=True, wide=20),
        # One new token for each of 64 sequences.
        dict(name="append_rope_64", kind="append", n_seq=64, q_lo=1, q_hi=1, c_lo=1, c_hi=4096, lens_seed=4, h_q=16, h_kv=2, d=256,
             page=16, rot=64, layout="halves", scaling="none", base=1e7, factor=1, norm=True),
        # Speculative decoding: four drafted tokens for each of 37 sequences.
        dict(name="append_rope_37x4", kind="append", n_seq=37, q_lo=4, q_hi=4, c_lo=100, c_hi=4000, lens_seed=5, h_q=32, h_kv=8, d=128,
             page=32, rot=128, layout="halves", scaling="linear", base=1e4, factor=8, norm=False),
        # Prompts of a prefill batch into fresh and half-filled pages.
        dict(name="append_rope_varlen_16", kind="append", n_seq=16, q_lo=1, q_hi=2048, c_lo=0, c_hi=100, lens_seed=6, h_q=16, h_kv=2,
             d=256, page=64, rot=64, layout="halves", scaling="none", base=1e7, factor=1, norm=True),
        # Four samples of one user's prompt. Latency.
        dict(name="shared_4", kind="shared", n_seq=4, n_groups=1, s_lo=1000, s_hi=1000, q_lo=1, q_hi=1, c_lo=1, c_hi=200, lens_seed=7,
             h_q=16, h_kv=2, d=256, page=16, gate=True),
        # A serving batch behind one long system prompt that ends inside a page.
        dict(name="shared_64", kind="shared", n_seq=64, n_groups=1, s_lo=8190, s_hi=8190, q_lo=1, q_hi=1, c_lo=0, c_hi=1000, lens_seed=8,
             h_q=16, h_kv=2, d=256, page=16, gate=True),
        # Samples of 24 prompts, four each.
        dict(name="shared_24x4", kind="shared", n_seq=96, n_groups=24, s_lo=300, s_hi=6000, q_lo=1, q_hi=1, c_lo=0, c_hi=600, lens_seed=9,
             h_q=32, h_kv=8, d=128, page=32, gate=False),
        # Drafts of a batch behind a shared prompt.
        dict(name="shared_drafts_37x4", kind="shared", n_seq=37, n_groups=1, s_lo=2049, s_hi=2049, q_lo=4, q_hi=4, c_lo=0, c_hi=500,
             lens_seed=10, h_q=32, h_kv=8, d=128, page=32, gate=False),
        # Many sequences behind a long document.
        dict(name="shared_128", kind="shared", n_seq=128, n_groups=1, s_lo=16384, s_hi=16384, q_lo=1, q_hi=1, c_lo=1, c_hi=2000, lens_seed=11,
             h_q=20, h_kv=4, d=128, page=64, gate=False),
        # Questions about one document, a prefill batch.
        dict(name="shared_questions_8", kind="shared", n_seq=8, n_groups=1, s_lo=6000, s_hi=6000, q_lo=1, q_hi=300, c_lo=0, c_hi=0, lens_seed=12,
             h_q=16, h_kv=4, d=128, page=64, gate=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    case = _drawn(rng)
    most = {"rope": (1e18, 6.7e7), "append": (1e18, 3.5e8), "shared": (6.5e10, 2.1e8)}[case["kind"]]       # of the largest listed
    while work(case)["flops"] > most[0] or work(case)["bytes"] > most[1]:
        for key in ("q_hi", "c_hi", "s_hi") if case["kind"] == "shared" else ("q_hi",):
            case[key] = -(-2 * case[key] // 3)
            case[key[0] + "_lo"] = min(case[key[0] + "_lo"], case[key])
        if case["kind"] == "append" and case["q_hi"] == 1:
            case["n_seq"] = -(-2 * case["n_seq"] // 3)
    return case


def _drawn_turn(rng, d):
    scaling = rng.choice(["none", "none", "linear", "parts"])
    return dict(rot=rng.choice([d, d, d // 2, d // 4, d // 4, d // 8, 2 * rng.randint(1, d // 2)]), layout=rng.choice(["halves", "halves", "pairs"]),
                scaling=scaling, base=rng.choice([1e4, 5e5, 1e7]), factor=1 if scaling == "none" else rng.choice([2, 4, 8, 40]),
                norm=rng.random() < 0.5)


def _drawn(rng):
    kind = rng.choice(["rope", "append", "append", "shared", "shared", "shared"])
    lens_seed = rng.randrange(1 << 16)
    if kind == "rope":
        d = rng.choice([64, 80, 96, 128, 128, 192, 256, 256])
        heads, turn = rng.choice([1, 2, 4, 8, 16, 16, 20, 32]), _drawn_turn(rng, d)
        wide = heads + rng.choice([0, 2, 4, 16])
        if rng.random() < 0.4:
            q = rng.choice([1, 1, rng.randint(2, 8)])
            return dict(kind=kind, n_seq=_log_int(rng, 1, 256), q_lo=q, q_hi=q, c_lo=0, c_hi=_log_int(rng, 16, 1000000), lens_seed=lens_seed,
                        heads=heads, d=d, wide=wide, **turn)
        n_seq = rng.choice([1, 1, rng.randint(2, 16)])
        q = _log_int(rng, 10, 2 ** 24 // (heads * d * n_seq))
        return dict(kind=kind, n_seq=n_seq, q_lo=q if n_seq == 1 else 1, q_hi=q, c_lo=0, c_hi=_log_int(rng, 16, 1000000), lens_seed=lens_seed,
                    heads=heads, d=d, wide=wide, **turn)
    heads, d = rng.choice([(2, 256), (2, 256), (1, 256), (8, 128), (4, 128), (2, 128), (8, 64)])
    group = rng.choice([8, 8, 4, 4, 5, 1, 16]) if d == 256 else rng.choice([4, 4, 8, 5, 1])
    more = dict(lens_seed=lens_seed, h_q=group * heads, h_kv=heads, d=d, page=rng.choice([16, 16, 32, 64]))
    if kind == "append":
        more.update(_drawn_turn(rng, d))
        if rng.random() < 0.5:
            q = rng.choice([1, 1, 1, rng.randint(2, 8)])
            return dict(kind=kind, n_seq=_log_int(rng, 1, 256), q_lo=q, q_hi=q, c_lo=0, c_hi=_log_int(rng, 16, 8192), **more)
        return dict(kind=kind, n_seq=rng.randint(1, 16), q_lo=1, q_hi=_log_int(rng, 10, 2048), c_lo=0, c_hi=100, **more)
    more["gate"] = rng.random() < 0.5
    q_lo, q_hi = rng.choice([(1, 1), (1, 1), (1, 1), (rng.randint(2, 8),) * 2, (1, _log_int(rng, 10, 300))])
    n_groups = rng.choice([1, 1, 1, rng.randint(2, 24)])
    each = _log_int(rng, 2, 128 if n_groups == 1 else 8)
    if q_hi > 8:
        each = min(each, 12)
    s_hi = _log_int(rng, 30, 16384)
    s_lo = s_hi if n_groups == 1 else rng.randint(1, s_hi)
    return dict(kind=kind, n_seq=n_groups * each, n_groups=n_groups, s_lo=s_lo, s_hi=s_hi, q_lo=q_lo, q_hi=q_hi, c_lo=0,
                c_hi=_log_int(rng, 16, 2000), **more)


def _lens(case):
    """(new tokens, tokens in all, shared tokens) of each sequence."""
    r = random.Random(case["lens_seed"])
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["n_seq"])]
    kv = [r.randint(case["c_lo"], case["c_hi"]) + n for n in q]
    if case["kind"] != "shared":
        return q, kv, None
    shared = [r.randint(case["s_lo"], case["s_hi"]) for _ in range(case["n_groups"])]
    shared = [n for n in shared for _ in range(case["n_seq"] // case["n_groups"])]
    return q, [n + m for n, m in zip(kv, shared)], shared


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


def _turning(case, g):
    """Frequencies [rot / 2], the factor of cosine and sine, and the norms of keys and queries."""
    i = torch.arange(case["rot"] // 2, dtype=torch.float64)
    freq, factor = case["base"] ** (-2 * i / case["rot"]), case["factor"]
    amplitude = 1.0
    if case["scaling"] == "linear":
        freq = freq / factor
    elif case["scaling"] == "parts":                      # trained on 32,768 tokens: waves that went round 32 times are kept
        turns = 32768 * freq / (2 * math.pi)
        keep = ((turns - 1) / 31).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
        amplitude = 0.1 * math.log(factor) + 1
    norms = [g.normal(case["d"], std=0.2, dtype=torch.float32) if case["norm"] else None for _ in "kq"]
    return dict(freq=freq.float().cuda(), amplitude=amplitude, norm_k=norms[0], norm_q=norms[1])


def _cache(case, g, kv, shared):
    """The cache with every page's codes and scales filled, and a table of pages in no order. A group's whole shared pages are
    the same ones for its sequences; the page in which the shared tokens end is each sequence's own, a copy of the first's."""
    page, h, d = case["page"], case["h_kv"], case["d"]
    each = len(kv) // case["n_groups"] if shared else 1
    width = max(-(-n // page) for n in kv) + 1
    rows, at, copies = [], 0, []
    for b, n in enumerate(kv):
        first = rows[b - b % each] if b % each else []
        common = shared[b] // page if first else 0
        own_pages = -(-n // page) - common
        row = first[:common] + list(range(at, at + own_pages))
        if first and shared[b] % page:
            copies.append((first[common], at))
        at += own_pages
        rows.append(row)
    order = g.order(at + 7)
    flat = torch.full((len(kv), width), -1, dtype=torch.int32)
    for b, row in enumerate(rows):
        flat[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
    flat = flat.cuda()
    table = torch.where(flat >= 0, order[flat.clamp(min=0).long()].to(torch.int32), -1)
    s = dict(k=g.codes(at + 7, h, page, d), v=g.codes(at + 7, h, d, page), k_scale=g.scales(at + 7, h),
             v_scale=g.scales(at + 7, h), table=table, width=width)
    if copies:
        a, b = order[torch.tensor(copies, device="cuda").T]
        for name in ("k", "v", "k_scale", "v_scale"):
            s[name][b] = s[name][a]
    return s


def prepare(case, seed):
    g = _Gen(seed)
    q, kv, shared = _lens(case)
    d, T = case["d"], sum(q)
    s = dict(case=case, q_len=_ints(q), cu=_ints(_cumulative(q)), kv_len=_ints(kv), T=T)
    if case["kind"] == "rope":
        # The rows of a fused projection, of which these heads are the first.
        rows = g.normal(T, case["wide"] * d)
        s.update(_turning(case, g), x=rows[:, :case["heads"] * d].view(T, case["heads"], d),
                 y=torch.empty(T, case["heads"], d, dtype=torch.bfloat16, device="cuda"))
    else:
        h, h_q, page = case["h_kv"], case["h_q"], case["page"]
        s.update(_cache(case, g, kv, shared))
        if case["kind"] == "append":
            # Queries, keys and values as slices of one projection's rows. Some tokens are larger than what their page holds.
            rows = g.normal(T, (h_q + 2 * h) * d) * (1 + g.normal(T, 1, std=0.3).abs())
            s.update(_turning(case, g), q=rows[:, :h_q * d].view(T, h_q, d), new_k=rows[:, h_q * d:(h_q + h) * d].view(T, h, d),
                     new_v=rows[:, (h_q + h) * d:].view(T, h, d), q_out=torch.empty(T, h_q, d, dtype=torch.bfloat16, device="cuda"))
            # Pages are read back from the start of the first one that changes.
            back = [n - (n - m) // page * page for m, n in zip(q, kv)]
            s.update(back=_ints(back), back_cu=_ints(_cumulative(back)), back_T=sum(back),
                     out_k=torch.empty(sum(back), h, d, dtype=torch.bfloat16, device="cuda"),
                     out_v=torch.empty(sum(back), h, d, dtype=torch.bfloat16, device="cuda"))
        else:
            each = case["n_seq"] // case["n_groups"]
            s.update(q=g.normal(T, h_q, d, std=2.0), o=torch.empty(T, h_q, d, dtype=torch.bfloat16, device="cuda"),
                     gate=g.normal(T, h_q, d) if case["gate"] else None, max_q=max(q), max_kv=max(kv), scale=d ** -0.5,
                     groups=_ints([each * i for i in range(case["n_groups"] + 1)]), shared=_ints(shared[::each]))
    if own:                                      # the descriptions and workspace that a program keeps beside its cache
        import baloon_amd as bx
        if case["kind"] != "rope":
            s["cache"] = bx.kv8_cache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if case["kind"] == "shared":
            n = bx.ix_kv8_attn_shared_workspace_size(s["cache"], case["n_seq"], T, s["max_q"], case["n_groups"], case["h_q"])
            s["ws"] = torch.zeros(max(n, 1), dtype=torch.uint8, device="cuda")
        else:
            layout = bx.ROPE_PAIRS if case["layout"] == "pairs" else bx.ROPE_HALVES
            s["rope_k"], s["rope_q"] = (bx.rope(s["freq"], layout, s["amplitude"], s[n], 1.0, EPS) for n in ("norm_k", "norm_q"))
    return s


# ---------------------------------------------------------------------------------------------
# The library's calls
# ---------------------------------------------------------------------------------------------

def _run_own(s):
    import baloon_amd as bx
    c = s["case"]
    if c["kind"] == "rope":
        bx.check("ix_rope_rows", bx.ix_rope_rows(s["rope_q"], c["n_seq"], s["T"], s["cu"], s["kv_len"], s["x"], c["heads"], c["d"], s["y"]))
        return dict(y=s["y"])
    if c["kind"] == "append":
        bx.check("ix_kv8_append_rope", bx.ix_kv8_append_rope(s["cache"], c["n_seq"], s["T"], s["cu"], s["kv_len"], s["table"], s["width"],
                                                             s["new_k"], s["new_v"], s["rope_k"], s["q"], c["h_q"], s["rope_q"], s["q_out"]))
        bx.check("ix_kv8_read", bx.ix_kv8_read(s["cache"], c["n_seq"], s["back_T"], s["back_cu"], s["kv_len"], s["table"],
                                               s["width"], s["out_k"], s["out_v"]))
        return dict(q=s["q_out"], k=s["out_k"], v=s["out_v"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    bx.check("ix_kv8_attn_shared", bx.ix_kv8_attn_shared(s["cache"], c["n_seq"], s["T"], s["max_q"], s["cu"], s["kv_len"], s["table"],
                                                         s["width"], c["n_groups"], s["groups"], s["shared"], s["q"], c["h_q"], s["scale"],
                                                         s["gate"], s["o"], s["ws"], s["ws"].numel()))
    return dict(o=s["o"])


# ---------------------------------------------------------------------------------------------
# The plain form
# ---------------------------------------------------------------------------------------------

def _tokens(lens, cu, T):
    """(sequence, place in it) of each of T packed rows."""
    b = torch.repeat_interleave(torch.arange(lens.numel(), device="cuda"), lens.long(), output_size=T)
    return b, torch.arange(T, device="cuda") - cu.long()[b]


def _turned(s, x, norm):
    """Rows x [T][heads][d] normed and turned, rounded to bf16. The angles, up to a million turns, are in 64 bits."""
    c, x = s["case"], x.float()
    if norm is not None:
        x = x * (1.0 / torch.sqrt((x * x).mean(2, keepdim=True) + EPS)) * (norm + 1.0)
    b, i = _tokens(s["q_len"], s["cu"], s["T"])
    pos = (s["kv_len"] - s["q_len"]).long()[b] + i
    angle = pos.double()[:, None] * s["freq"].double()
    cos, sin = ((f(angle) * s["amplitude"]).float()[:, None] for f in (torch.cos, torch.sin))
    rot = c["rot"]
    if c["layout"] == "halves":
        lo, hi = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], 2)
    else:
        even, odd = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([even * cos - odd * sin, odd * cos + even * sin], 3).flatten(2)
    return torch.cat([turned, x[..., rot:]], 2).to(torch.bfloat16)


def _plain_rope(s):
    return dict(y=_turned(s, s["x"], s["norm_q"]))


def _plain_append(s):
    c, page = s["case"], s["case"]["page"]
    new_k, new_v = _turned(s, s["new_k"], s["norm_k"]), s["new_v"]
    table, kv = s["table"].long(), s["kv_len"].long()
    b, i = _tokens(s["q_len"], s["cu"], s["T"])
    first = kv - s["q_len"]
    pos = first[b] + i
    at, slot = table[b, pos // page], pos % page
    # the first page of each sequence may hold older tokens, in its first `held` slots
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
        quantum = scale[at][:, :, None]
        return torch.where(quantum > 0, torch.round(x.float() / quantum), 0.0).clamp(-127, 127).to(torch.int8)

    now_k, r_k = grow(new_k, s_k)
    now_v, r_v = grow(new_v, s_v)
    old_k, old_v = s["k"][p0], s["v"][p0]
    s["k"][p0] = torch.where(older[:, None, :, None], torch.round(old_k.float() * r_k[:, :, None, None]).to(torch.int8), old_k)
    s["v"][p0] = torch.where(older[:, None, None, :], torch.round(old_v.float() * r_v[:, :, None, None]).to(torch.int8), old_v)
    heads = torch.arange(c["h_kv"], device="cuda")[None, :]
    s["k"][at[:, None], heads, slot[:, None]] = codes(new_k, now_k)
    s["v"][at[:, None], heads, :, slot[:, None]] = codes(new_v, now_v)
    s_k.copy_(now_k)
    s_v.copy_(now_v)
    # and back
    b, i = _tokens(s["back"], s["back_cu"], s["back_T"])
    pos = (kv - s["back"])[b] + i
    at, slot = table[b, pos // page][:, None], (pos % page)[:, None]
    k = s["k"][at, heads, slot].float() * s_k[at, heads][:, :, None]
    v = s["v"][at, heads, :, slot].float() * s_v[at, heads][:, :, None]
    return dict(q=_turned(s, s["q"], s["norm_q"]), k=k.to(torch.bfloat16), v=v.to(torch.bfloat16), k_scale=s_k, v_scale=s_v)


def _plain_shared(s):
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
    seen = ((j <= pos) & (j < kv[:, None, None])).repeat_interleave(G, 1)[:, None]
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
    return {"rope": _plain_rope, "append": _plain_append, "shared": _plain_shared}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------

def work(case):
    q, kv, shared = _lens(case)
    d, T = case["d"], sum(q)
    turn = 3 * case.get("rot", 0) + (4 * d if case.get("norm") else 0)          # operations of a head's row
    if case["kind"] == "rope":
        return dict(bytes=4 * T * case["heads"] * d, flops=T * case["heads"] * turn)
    h, page = case["h_kv"], case["page"]
    if case["kind"] == "append":
        back = sum(n - (n - m) // page * page for m, n in zip(q, kv))
        # rows in, codes and turned queries out; codes in, rows back out
        return dict(bytes=2 * h * d * (3 * T + 3 * back) + 4 * T * case["h_q"] * d,
                    flops=2 * h * d * (4 * T + back) + T * (h + case["h_q"]) * turn)
    each = case["n_seq"] // case["n_groups"]
    pairs = sum(m * n - m * (m - 1) // 2 for m, n in zip(q, kv))
    tokens = sum(n - m for n, m in zip(kv, shared)) + sum(shared[::each])
    rows = T * case["h_q"] * d
    return dict(bytes=2 * tokens * h * d + 2 * rows * (3 if case["gate"] else 2), flops=4 * pairs * case["h_q"] * d)


# ---------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------------

def _exact_turn(s, x, norm, q, kv):
    """Rows x in 64 bits as complex numbers times amplitude * exp(1j * angle); the rounding to bf16 is the caller's."""
    c, x = s["case"], x.to(torch.float64)
    if norm is not None:
        x = x / torch.sqrt(x.square().sum(2, keepdim=True) / c["d"] + EPS) * (1.0 + norm.to(torch.float64))
    pos = torch.cat([torch.arange(n - m, n, dtype=torch.float64) for m, n in zip(q, kv)]).cuda()
    angle = torch.outer(pos, s["freq"].to(torch.float64))
    by = torch.polar(torch.full_like(angle, s["amplitude"]), angle)[:, None, :]
    part = x[..., :c["rot"]]
    if c["layout"] == "halves":
        z = torch.complex(*part.chunk(2, dim=2)) * by
        part = torch.cat((z.real, z.imag), dim=2)
    else:
        part = torch.view_as_real(torch.view_as_complex(part.unflatten(2, (-1, 2)).contiguous()) * by).flatten(2)
    return torch.cat((part, x[..., c["rot"]:]), dim=2)


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    q, kv, _ = _lens(case)
    if case["kind"] == "rope":
        return dict(y=_exact_turn(s, s["x"], s["norm_q"], q, kv))
    h, d, page = case["h_kv"], case["d"], case["page"]
    cu = _cumulative(q)
    table = s["table"].cpu().tolist()
    if case["kind"] == "append":
        rows = dict(k=_exact_turn(s, s["new_k"], s["norm_k"], q, kv).to(torch.bfloat16), v=s["new_v"])   # turned keys are held in bf16
        out = {"k": [], "v": []}
        scale = {"k": s["k_scale"].to(f64), "v": s["v_scale"].to(f64)}
        for b in range(case["n_seq"]):
            first, row = kv[b] - q[b], cu[b]
            for p in range(first // page, -(-kv[b] // page)):
                at, lo, hi = table[b][p], max(first, p * page), min(kv[b], (p + 1) * page)
                held, new = lo - p * page, hi - lo
                for name in ("k", "v"):
                    x = rows[name][row:row + new].to(f64).transpose(0, 1)                   # [h, new, d]
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
        return dict(q=_exact_turn(s, s["q"], s["norm_q"], q, kv), k=torch.cat(out["k"]), v=torch.cat(out["v"]), k_scale=scale["k"],
                    v_scale=scale["v"])
    G = case["h_q"] // h
    o = torch.zeros(sum(q), case["h_q"], d, dtype=f64, device="cuda")
    for b in range(case["n_seq"]):
        pages = s["table"][b, :-(-kv[b] // page)].long()
        hidden = torch.arange(kv[b], device="cuda")[None, :] > torch.arange(kv[b] - q[b], kv[b], device="cuda")[:, None]
        for e in range(h):
            k = (s["k"][pages, e].to(f64) * s["k_scale"][pages, e].to(f64)[:, None, None]).reshape(-1, d)[:kv[b]]
            v = (s["v"][pages, e].to(f64) * s["v_scale"][pages, e].to(f64)[:, None, None]).transpose(1, 2).reshape(-1, d)[:kv[b]]
            x = s["q"][cu[b]:cu[b + 1], e * G:(e + 1) * G].to(f64)                          # [q, G, d]
            a = ((x.reshape(-1, d) @ k.T) * s["scale"]).masked_fill(hidden.repeat_interleave(G, 0), float("-inf"))
            o[cu[b]:cu[b + 1], e * G:(e + 1) * G] = (torch.softmax(a, 1) @ v).view(-1, G, d)
    if s["gate"] is not None:
        o = o * torch.sigmoid(s["gate"].to(f64))
    return dict(o=o)
