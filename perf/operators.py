"""Timed and checked cases of the paged-cache operators.

Four calls of the package, each beside its plain form in elementary torch operations:

  append   paged_append              QK-norm, rotary positions, k and v written into pages
  decode   paged_attention_decode    one new token per sequence over the pages
  packed   attention_prompt          whole prompts, causal, packed, K and V packed beside q
  paged    paged_attention_prompt    prompts whose K and V lie in pages, after a cached prefix
"""
import random

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
THETA = 1e6  # the rotary base of this framework's shapes


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the attention block's entry in one decode step of 64 sessions, 4B shape, fp32 rows from the matmuls
        dict(name="append-64-sessions", op="append", n_seqs=64, new_lo=1, new_hi=1, pre_lo=1024, pre_hi=1151, heads=32, kv=8, hd=128,
             page=64, cache="bf16", inp="f32", norm=True, rope=True, hnd=False, fused=False, empty=0, lens_seed=1),
        # a 4096-token prompt entering the cache, 8B shape
        dict(name="append-4096-prompt", op="append", n_seqs=1, new_lo=4096, new_hi=4096, pre_lo=0, pre_hi=0, heads=32, kv=8, hd=128,
             page=64, cache="bf16", inp="f32", norm=True, rope=True, hnd=False, fused=False, empty=0, lens_seed=2),
        # ragged prompts from one fused 16-bit projection, no QK-norm, head-major pages
        dict(name="append-ragged-fused", op="append", n_seqs=13, new_lo=1, new_hi=1500, pre_lo=0, pre_hi=700, heads=12, kv=4, hd=64,
             page=32, cache="f16", inp="f16", norm=False, rope=True, hnd=True, fused=True, empty=0, lens_seed=3),
        # the smallest call: one short conversation of the 1.7B shape
        dict(name="decode-1x33", op="decode", n_seqs=1, len_lo=33, len_hi=33, heads=16, kv=8, hd=128, page=16, cache="f16", hnd=False,
             empty=0, lens_seed=4),
        # one long conversation of the 8B shape, decoding after its 4096-token prompt: few rows, long axis
        dict(name="decode-1x4200", op="decode", n_seqs=1, len_lo=4200, len_hi=4200, heads=32, kv=8, hd=128, page=64, cache="bf16", hnd=False,
             empty=0, lens_seed=5),
        # 64 sessions at about 1024 positions, 4B shape
        dict(name="decode-64x1100", op="decode", n_seqs=64, len_lo=1025, len_hi=1152, heads=32, kv=8, hd=128, page=64, cache="bf16", hnd=False,
             empty=0, lens_seed=6),
        # 128 sessions of every length up to the shapes' context of 8192
        dict(name="decode-128-ragged", op="decode", n_seqs=128, len_lo=1, len_hi=8192, heads=32, kv=8, hd=128, page=128, cache="bf16", hnd=True,
             empty=0, lens_seed=7),
        # heads of 64 without groups, slots that hold no sequence yet
        dict(name="decode-48-hd64", op="decode", n_seqs=48, len_lo=1, len_hi=3000, heads=12, kv=12, hd=64, page=16, cache="f16", hnd=False,
             empty=5, lens_seed=8),
        # a 512-token prompt, 4B shape
        dict(name="packed-512", op="packed", n_seqs=1, new_lo=512, new_hi=512, heads=32, kv=8, hd=128, cache="bf16", fused=True, empty=0,
             lens_seed=9),
        # prompts of very different lengths in one call, 1.7B shape
        dict(name="packed-ragged", op="packed", n_seqs=9, new_lo=1, new_hi=4096, heads=16, kv=8, hd=128, cache="f16", fused=False, empty=4,
             lens_seed=10),
        # one prompt as long as the shapes' context
        dict(name="packed-8192", op="packed", n_seqs=1, new_lo=8192, new_hi=8192, heads=32, kv=8, hd=128, cache="bf16", fused=False, empty=0,
             lens_seed=11),
        # 16 sessions continue a shared 256-token prefix up to 1024 positions, 4B shape
        dict(name="paged-16x768", op="paged", n_seqs=16, new_lo=700, new_hi=768, pre_lo=256, pre_hi=256, heads=32, kv=8, hd=128, page=64,
             cache="bf16", hnd=False, empty=0, lens_seed=12),
    ]


def log_int(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    heads, kv = rng.choice([(16, 8), (32, 8), (32, 4), (8, 8), (12, 4), (12, 12), (5, 1), (16, 1)])
    hd = rng.choice([64, 128, 128])
    c = dict(op=rng.choice(["append", "decode", "packed", "paged"]), heads=heads, kv=kv, hd=hd, cache=rng.choice(["f16", "bf16"]),
             empty=rng.choice([0, 0, 3, 5]), lens_seed=rng.randrange(1 << 20))
    if c["op"] != "packed":
        c["page"], c["hnd"] = rng.choice([16, 32, 64, 128, 256]), rng.random() < 0.5
    if c["op"] == "append":
        c["n_seqs"] = log_int(rng, 1, 128)
        top = log_int(rng, 1, 4096 // c["n_seqs"]) if c["n_seqs"] < 4096 else 1
        c["new_lo"], c["new_hi"] = rng.choice([1, max(1, top // 2), top]), top
        c["pre_lo"], c["pre_hi"] = 0, log_int(rng, 1, 2000)
        c["inp"], c["norm"], c["rope"] = rng.choice(["f32", "f32", c["cache"]]), rng.random() < 0.6, rng.random() < 0.8
        c["fused"] = rng.random() < 0.5
    elif c["op"] == "decode":
        c["n_seqs"] = log_int(rng, 1, 128)
        c["len_hi"] = log_int(rng, 1, 8192)
        c["len_lo"] = rng.choice([1, max(1, c["len_hi"] // 2), c["len_hi"]])
        if c["kv"] > 8:  # no more work than the largest listed case
            c["len_hi"] = min(c["len_hi"], 5000)
            c["len_lo"] = min(c["len_lo"], c["len_hi"])
    else:
        top = log_int(rng, 1, 6000)
        c["n_seqs"] = log_int(rng, 1, max(1, min(64, 24_000_000 // (top * top))))
        c["new_lo"], c["new_hi"] = rng.choice([1, max(1, top // 2), top]), top
        c["fused"] = rng.random() < 0.5
        if c["op"] == "paged":
            del c["fused"]
            c["pre_lo"], c["pre_hi"] = 0, log_int(rng, 1, max(1, min(2000, 24_000_000 // (top * c["n_seqs"]) - top, 8192 - top)))
    return c


def lengths(c):
    """New tokens and cache lengths (the new ones included) of each sequence; the case's alone, whatever the seed."""
    r, new, total = random.Random(c["lens_seed"]), [], []
    for s in range(c["n_seqs"]):
        gone = c["empty"] and s % c["empty"] == c["empty"] - 1
        if c["op"] == "decode":
            new.append(1)
            total.append(0 if gone else r.randint(c["len_lo"], c["len_hi"]))
        else:
            n = 0 if gone else r.randint(c["new_lo"], c["new_hi"])
            new.append(n)
            total.append(n + (r.randint(c["pre_lo"], c["pre_hi"]) if "pre_lo" in c else 0))
    return new, total


def work(c):
    new, total = lengths(c)
    n, io = sum(new), c["heads"] * c["hd"]
    if c["op"] == "append":
        row = (c["heads"] + 2 * c["kv"]) * c["hd"]
        size = 4 if c["inp"] == "f32" else 2
        return {"bytes": n * (row * (size + 2) + (c["hd"] * 4 if c["rope"] else 0)), "flops": 8 * n * row}
    # token i of n ends at position total - n + i; it sees that many keys and itself
    pairs = sum(total) if c["op"] == "decode" else sum(m * (t - m) + m * (m + 1) // 2 for m, t in zip(new, total))
    return {"bytes": 2 * 2 * n * io + 2 * 2 * sum(total) * c["kv"] * c["hd"], "flops": 4 * pairs * io}


# ----------------------------------------------------------------- inputs
def rope_table(n, hd, device):
    """[n][hd/2 cosines | hd/2 sines], angles in 64 bits, rounded once."""
    inv = THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=device) / hd)
    ang = torch.arange(n, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def prepare(case, seed):
    c = case
    dev, dt = "cuda", DTYPE[c["cache"]]
    gen = torch.Generator(device=dev).manual_seed(seed)

    def rand(*shape, dtype=dt):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dtype)

    new, total = lengths(c)
    n, H, KV, D = sum(new), c["heads"], c["kv"], c["hd"]
    st = {"op": c["op"], "cache_dtype": dt, "heads": H, "kv": KV, "hd": D}
    # plans of the plain forms: where each new token lies in a padded [sequence, place] layout
    seq_of = [s for s, m in enumerate(new) for _ in range(m)]
    place = [i for m in new for i in range(m)]
    st["seq_of"] = torch.tensor(seq_of, dtype=torch.int64, device=dev)
    st["place"] = torch.tensor(place, dtype=torch.int64, device=dev)
    st["pos"] = torch.tensor([total[s] - new[s] + i for s, i in zip(seq_of, place)], dtype=torch.int64, device=dev)
    st["new"] = torch.tensor(new, dtype=torch.int32, device=dev)
    st["lens"] = torch.tensor(total, dtype=torch.int32, device=dev)
    st["max_new"], st["max_len"], st["n"] = max(new), max(1, max(total)), n
    cu = [0]
    for m in new:
        cu.append(cu[-1] + m)
    st["cu"] = torch.tensor(cu, dtype=torch.int32, device=dev)
    if c["op"] == "packed":
        if c["fused"]:  # rows of one projection
            qkv = rand(n, H + 2 * KV, D)
            st["q"], st["k"], st["v"] = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
        else:
            st["q"], st["k"], st["v"] = rand(n, H, D), rand(n, KV, D), rand(n, KV, D)
        return st
    page = c["page"]
    need = [-(-t // page) for t in total]
    width = max(1, max(need))
    pages = sum(need) + 3  # a pool with a few pages to spare, the sequences' pages all over it
    shape = (pages, KV, page, D) if c["hnd"] else (pages, page, KV, D)
    k, v = rand(*shape), rand(*shape)  # stale values of earlier conversations where nothing was written yet
    st["k"], st["v"] = (k.transpose(1, 2), v.transpose(1, 2)) if c["hnd"] else (k, v)
    perm = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    first = torch.tensor([0] + need, device=dev).cumsum(0)[:-1]
    at = first[:, None] + torch.arange(width, device=dev)
    held = torch.arange(width, device=dev) < torch.tensor(need, device=dev)[:, None]
    st["table"] = torch.where(held, perm[at.clamp(max=pages - 1)], 0).to(torch.int32).contiguous()
    if c["op"] == "append":
        it = DTYPE[c["inp"]]
        if c["fused"]:
            qkv = rand(n, H + 2 * KV, D, dtype=it)
            st["q"], st["k_new"], st["v_new"] = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
        else:
            st["q"], st["k_new"], st["v_new"] = rand(n, H, D, dtype=it), rand(n, KV, D, dtype=it), rand(n, KV, D, dtype=it)
        st["q_norm"] = 1 + 0.1 * rand(D, dtype=torch.float32) if c["norm"] else None
        st["k_norm"] = 1 + 0.1 * rand(D, dtype=torch.float32) if c["norm"] else None
        st["rope"] = rope_table(max(total) + 1, D, dev) if c["rope"] else None
    else:
        st["q"] = rand(n, H, D)
    if own:
        import rpgbarengine_b200 as rb
        st["pool"] = rb.PagedKV(st["k"], st["v"])
        st["batch"] = rb.PagedBatch(st["table"], st["lens"], cu_q=None if c["op"] == "decode" else st["cu"], n_tokens=n)
    return st


# ------------------------------------------------------------ plain forms
def norm_rope_plain(x, gain, rope, pos):
    x = x.float()
    if gain is not None:
        x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * gain
    if rope is not None:
        h = x.shape[-1] // 2
        c, s = rope[pos, None, :h], rope[pos, None, h:]
        a, b = x[..., :h], x[..., h:]
        x = torch.cat([a * c - b * s, b * c + a * s], -1)
    return x


def softmax_plain(s, seen):
    """Softmax over the last axis of the places that are seen; zeros where none is."""
    s = s.masked_fill(~seen, float("-inf"))
    m = s.amax(-1, keepdim=True)
    e = (s - torch.where(m > float("-inf"), m, 0.0)).exp()
    return e / e.sum(-1, keepdim=True).clamp(min=1e-30)


def gather_pages(pool, table, n):
    """[sequence, kv head, place, dim] in 32 bits."""
    x = pool[table.long()]  # [sequence, page, slot, kv head, dim]
    x = x.reshape(table.shape[0], -1, x.shape[-2], x.shape[-1])
    return x[:, :n].permute(0, 2, 1, 3).float()


def attend_plain(st, k, v, first):
    """q's rows over padded k, v [sequence, kv head, place, dim]; `first`: each sequence's position of its row 0."""
    S, KV, L, D = k.shape
    G, dev = st["heads"] // KV, k.device
    q = torch.zeros(S, st["max_new"], KV * G, D, device=dev)
    q[st["seq_of"], st["place"]] = st["q"].float()
    q = q.view(S, -1, KV, G, D).permute(0, 2, 3, 1, 4).reshape(S, KV, -1, D)  # rows: (head of the group, token)
    s = (q @ k.transpose(-1, -2) * D ** -0.5).view(S, KV, G, -1, L)
    t = torch.arange(L, device=dev)
    last = first[:, None] + torch.arange(st["max_new"], device=dev)
    seen = (t <= last[..., None]) & (t < st["lens"][:, None, None])
    p = softmax_plain(s, seen[:, None, None])
    o = p.view(S, KV, -1, L) @ v
    o = o.view(S, KV, G, -1, D).permute(0, 3, 1, 2, 4).reshape(S, -1, KV * G, D)
    return o[st["seq_of"], st["place"]].to(st["cache_dtype"])


def run_plain(st):
    if st["op"] == "append":
        q = norm_rope_plain(st["q"], st["q_norm"], st["rope"], st["pos"]).to(st["cache_dtype"])
        k = norm_rope_plain(st["k_new"], st["k_norm"], st["rope"], st["pos"]).to(st["cache_dtype"])
        size = st["k"].shape[1]
        page, slot = st["table"][st["seq_of"], st["pos"] // size].long(), st["pos"] % size
        st["k"][page, slot] = k
        st["v"][page, slot] = st["v_new"].to(st["cache_dtype"])
        return {"q": q, "k": st["k"], "v": st["v"]}
    first = (st["lens"] - st["new"]).long()
    if st["op"] == "packed":
        S, L = st["new"].numel(), st["max_new"]
        k = torch.zeros(S, L, st["kv"], st["hd"], device=st["k"].device)
        v = torch.zeros_like(k)
        k[st["seq_of"], st["place"]] = st["k"].float()
        v[st["seq_of"], st["place"]] = st["v"].float()
        return {"out": attend_plain(st, k.transpose(1, 2), v.transpose(1, 2), first)}
    k, v = gather_pages(st["k"], st["table"], st["max_len"]), gather_pages(st["v"], st["table"], st["max_len"])
    return {"out": attend_plain(st, k, v, first)}


def run(state):
    st = state
    if not own:
        return run_plain(st)
    import rpgbarengine_b200 as rb
    if st["op"] == "append":
        q = rb.paged_append(st["pool"], st["batch"], st["q"], st["k_new"], st["v_new"], q_norm=st["q_norm"], k_norm=st["k_norm"],
                            eps=EPS, rope=st["rope"])
        return {"q": q, "k": st["k"], "v": st["v"]}
    if st["op"] == "decode":
        return {"out": rb.paged_attention_decode(st["pool"], st["batch"], st["q"])}
    if st["op"] == "paged":
        return {"out": rb.paged_attention_prompt(st["pool"], st["batch"], st["q"])}
    return {"out": rb.attention_prompt(st["q"], st["k"], st["v"], st["cu"])}


# --------------------------------------------------------------- 64 bits
def exact(case, seed):
    """From the definitions, a sequence and a head at a time, in 64 bits."""
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    new, total = lengths(case)
    D, G = case["hd"], case["heads"] // case["kv"]
    size = case.get("page", 0)

    def rows_of(s, count):
        p = torch.arange(count, device="cuda")
        return st["table"][s].long()[p // size], p % size

    if case["op"] == "append":
        def turned(x, gain):
            x = x.double()
            if gain is not None:
                x = x / ((x * x).sum(-1, keepdim=True) / D + EPS).sqrt() * gain.double()
            if st["rope"] is None:
                return x
            cos, sin = st["rope"].double()[st["pos"]].chunk(2, -1)
            z = torch.complex(x[..., : D // 2], x[..., D // 2:]) * torch.complex(cos, sin)[:, None]
            return torch.cat([z.real, z.imag], -1)

        k, v = st["k"].double(), st["v"].double()
        k_new, v_new, at = turned(st["k_new"], st["k_norm"]), st["v_new"].double(), 0
        for s, m in enumerate(new):
            if m:
                pg, sl = (x[total[s] - m:] for x in rows_of(s, total[s]))
                k[pg, sl], v[pg, sl] = k_new[at:at + m], v_new[at:at + m]
            at += m
        return {"q": turned(st["q"], st["q_norm"]), "k": k, "v": v}
    out, at = torch.zeros(st["n"], case["heads"], D, dtype=torch.float64, device="cuda"), 0
    for s, (m, t) in enumerate(zip(new, total)):
        if m and t:
            ks, vs = (st["k"][at:at + m], st["v"][at:at + m]) if case["op"] == "packed" else (x[rows_of(s, t)] for x in (st["k"], st["v"]))
            for h in range(case["heads"]):
                kk, vv = ks[:, h // G].double(), vs[:, h // G].double()
                a = st["q"][at:at + m, h].double() @ kk.T / D ** 0.5
                a = a.masked_fill(torch.ones_like(a, dtype=torch.bool).triu(t - m + 1), float("-inf"))
                out[at:at + m, h] = torch.softmax(a, -1) @ vv
        at += m
    return {"out": out}
