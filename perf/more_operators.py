"""Timed and checked cases of the 8-bit paged cache and of shared prefixes.

Four calls of the package, each beside its plain form in elementary torch operations:

  append8  paged_append on a PagedKV8            QK-norm, rotary positions, k and v written as e4m3 with a scale a row
  decode8  paged_attention_decode on a PagedKV8  one new token per sequence over 8-bit pages
  read8    paged_read                            positions of 8-bit pages back into 16-bit pages
  shared   paged_attention_decode with a prefix  one new token per sequence; groups of sequences share their first positions
"""
import random

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn
TOP = 448.0  # the largest e4m3 value
EPS = 1e-6
THETA = 1e6  # the rotary base of this framework's shapes


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the attention block's entry in one decode step of 64 sessions, 4B shape, fp32 rows from the matmuls
        dict(name="append8-64-sessions", op="append8", n_seqs=64, new_lo=1, new_hi=1, pre_lo=1024, pre_hi=1151, heads=32, kv=8, hd=128,
             page=64, io="bf16", inp="f32", norm=True, rope=True, hnd=False, fused=False, empty=0, lens_seed=1),
        # a 4096-token prompt entering the cache, 8B shape
        dict(name="append8-4096-prompt", op="append8", n_seqs=1, new_lo=4096, new_hi=4096, pre_lo=0, pre_hi=0, heads=32, kv=8, hd=128,
             page=64, io="bf16", inp="f32", norm=True, rope=True, hnd=False, fused=False, empty=0, lens_seed=2),
        # ragged prompts from one fused 16-bit projection, no QK-norm, head-major pages
        dict(name="append8-ragged-fused", op="append8", n_seqs=13, new_lo=1, new_hi=1500, pre_lo=0, pre_hi=700, heads=12, kv=4, hd=64,
             page=32, io="f16", inp="f16", norm=False, rope=True, hnd=True, fused=True, empty=0, lens_seed=3),
        # the smallest call: one short conversation of the 1.7B shape
        dict(name="decode8-1x33", op="decode8", n_seqs=1, len_lo=33, len_hi=33, heads=16, kv=8, hd=128, page=16, io="f16", hnd=False,
             empty=0, lens_seed=4),
        # one long conversation of the 8B shape, decoding after its 4096-token prompt: few rows, long axis
        dict(name="decode8-1x4200", op="decode8", n_seqs=1, len_lo=4200, len_hi=4200, heads=32, kv=8, hd=128, page=64, io="bf16", hnd=False,
             empty=0, lens_seed=5),
        # 128 sessions of every length up to the shapes' context of 8192
        dict(name="decode8-128-ragged", op="decode8", n_seqs=128, len_lo=1, len_hi=8192, heads=32, kv=8, hd=128, page=128, io="bf16", hnd=True,
             empty=0, lens_seed=6),
        # heads of 64 without groups, slots that hold no sequence yet
        dict(name="decode8-48-hd64", op="decode8", n_seqs=48, len_lo=1, len_hi=3000, heads=12, kv=12, hd=64, page=16, io="f16", hnd=False,
             empty=5, lens_seed=7),
        # the shared 256-token opening of 64 sessions, read back for the prompts that continue it
        dict(name="read8-1x256", op="read8", n_seqs=1, len_lo=256, len_hi=256, kv=8, hd=128, page=64, to_page=64, io="bf16", hnd=False,
             empty=0, lens_seed=8),
        # conversations that were put aside in 8 bits and continue with a prompt of many tokens, pages of another size
        dict(name="read8-16x4096", op="read8", n_seqs=16, len_lo=1, len_hi=4096, kv=8, hd=128, page=64, to_page=16, io="f16", hnd=True,
             empty=0, lens_seed=9),
        # 64 sessions with a shared 256-token prefix at about 1024 positions, 4B shape
        dict(name="shared-64x256", op="shared", n_seqs=64, groups=1, loose=0, plen_lo=256, plen_hi=256, own_lo=700, own_hi=768, heads=32, kv=8,
             hd=128, page=64, io="bf16", cache="same", hnd=False, empty=0, lens_seed=10),
        # 256 short conversations over one opening as long as the shapes' context
        dict(name="shared-256x8192", op="shared", n_seqs=256, groups=1, loose=0, plen_lo=8192, plen_hi=8192, own_lo=1, own_hi=200, heads=32,
             kv=8, hd=128, page=128, io="bf16", cache="same", hnd=False, empty=0, lens_seed=11),
        # several characters' openings, the conversations' own positions in 8 bits, slots that hold no sequence yet
        dict(name="shared-groups-8bit", op="shared", n_seqs=45, groups=6, loose=2, plen_lo=100, plen_hi=3000, own_lo=1, own_hi=500, heads=16,
             kv=8, hd=128, page=32, io="f16", cache="e4m3", hnd=True, empty=7, lens_seed=12),
    ]


def log_int(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    heads, kv = rng.choice([(16, 8), (32, 8), (32, 4), (8, 8), (12, 4), (12, 12), (5, 1), (16, 1)])
    hd = rng.choice([64, 128, 128])
    c = dict(op=rng.choice(["append8", "decode8", "read8", "shared", "shared"]), heads=heads, kv=kv, hd=hd, io=rng.choice(["f16", "bf16"]),
             page=rng.choice([16, 32, 64, 128, 256]), hnd=rng.random() < 0.5, empty=rng.choice([0, 0, 3, 5]), lens_seed=rng.randrange(1 << 20))
    if c["op"] == "append8":
        c["n_seqs"] = log_int(rng, 1, 128)
        top = log_int(rng, 1, 4096 // c["n_seqs"])
        c["new_lo"], c["new_hi"] = rng.choice([1, max(1, top // 2), top]), top
        c["pre_lo"], c["pre_hi"] = 0, log_int(rng, 1, 2000)
        c["inp"], c["norm"], c["rope"] = rng.choice(["f32", "f32", c["io"]]), rng.random() < 0.6, rng.random() < 0.8
        c["fused"] = rng.random() < 0.5
    elif c["op"] == "shared":
        c["n_seqs"] = log_int(rng, 1, 256)
        c["groups"] = min(c["n_seqs"], log_int(rng, 1, 16))
        c["loose"] = rng.choice([0, 0, min(3, c["n_seqs"] - c["groups"])])
        wide = max(1.0, kv * hd / 1024)  # no more work than the largest listed case
        room = int(2_000_000 / wide / c["n_seqs"])
        c["plen_hi"] = log_int(rng, 1, max(1, min(8192, room // 2)))
        c["plen_lo"] = rng.choice([1, max(1, c["plen_hi"] // 2), c["plen_hi"]])
        c["own_hi"] = log_int(rng, 1, max(1, min(2000, room // 2, 300_000 // c["n_seqs"])))
        c["own_lo"] = rng.choice([1, max(1, c["own_hi"] // 2), c["own_hi"]])
        c["cache"] = rng.choice(["same", "e4m3"])
    else:
        c["n_seqs"] = log_int(rng, 1, 128 if c["op"] == "decode8" else 32)
        c["len_hi"] = log_int(rng, 1, 8192 if kv <= 8 else 5000)
        c["len_lo"] = rng.choice([1, max(1, c["len_hi"] // 2), c["len_hi"]])
        if c["op"] == "read8":
            del c["heads"]
            c["to_page"] = rng.choice([16, 32, 64, 128, 256])
    return c


def lengths(c):
    """New tokens, cache lengths (the new ones included), prefix lengths and the sequences' groups (-1: none); the case's alone, whatever
    the seed."""
    r, new, total = random.Random(c["lens_seed"]), [], []
    plen, group = [], [-1] * c["n_seqs"]
    if c["op"] == "shared":
        g, n = c["groups"], c["n_seqs"] - c["loose"]
        cuts = [0] + sorted(r.sample(range(1, n), g - 1)) + [n]
        plen = [r.randint(c["plen_lo"], c["plen_hi"]) for _ in range(g)]
        group = [max(k for k in range(g) if cuts[k] <= s) if s < n else -1 for s in range(c["n_seqs"])]
    for s in range(c["n_seqs"]):
        gone = c["empty"] and s % c["empty"] == c["empty"] - 1
        if c["op"] == "append8":
            n = 0 if gone else r.randint(c["new_lo"], c["new_hi"])
            new.append(n)
            total.append(n + r.randint(c["pre_lo"], c["pre_hi"]))
        elif c["op"] == "shared":
            n = r.randint(c["own_lo"], c["own_hi"])
            new.append(1)
            total.append(0 if gone else n + (plen[group[s]] if group[s] >= 0 else 0))
        else:
            n = r.randint(c["len_lo"], c["len_hi"])
            new.append(1)
            total.append(0 if gone else n)
    return new, total, plen, group


def work(c):
    new, total, plen, group = lengths(c)
    n, kv, hd = sum(new), c["kv"], c["hd"]
    row8, row16 = kv * (2 * hd + 8), kv * 4 * hd  # k and v of a position
    if c["op"] == "append8":
        row = (c["heads"] + 2 * kv) * hd
        size = 4 if c["inp"] == "f32" else 2
        return {"bytes": n * (row * size + c["heads"] * hd * 2 + row8 + (hd * 4 if c["rope"] else 0)), "flops": 10 * n * row}
    if c["op"] == "read8":
        return {"bytes": sum(total) * (row8 + row16), "flops": 2 * sum(total) * kv * hd}
    io = 2 * 2 * n * c["heads"] * hd
    flops = 4 * sum(total) * c["heads"] * hd
    if c["op"] == "decode8":
        return {"bytes": io + sum(total) * row8, "flops": flops}
    rest = sum(max(0, t - (plen[g] if g >= 0 else 0)) for t, g in zip(total, group))
    once = sum(p for k, p in enumerate(plen) if any(g == k and t for t, g in zip(total, group)))
    return {"bytes": io + once * row16 + rest * (row8 if c["cache"] == "e4m3" else row16), "flops": flops}


# ----------------------------------------------------------------- inputs
def rope_table(n, hd, device):
    """[n][hd/2 cosines | hd/2 sines], angles in 64 bits, rounded once."""
    inv = THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=device) / hd)
    ang = torch.arange(n, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c = case
    dev, dt = "cuda", DTYPE[c["io"]]
    gen = torch.Generator(device=dev).manual_seed(seed)

    def rand(*shape, dtype=dt):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dtype)

    new, total, plen, group = lengths(c)
    n, KV, D, page = sum(new), c["kv"], c["hd"], c["page"]
    st = {"op": c["op"], "io": dt, "kv": KV, "hd": D, "page": page, "n": n, "max_len": max(1, max(total))}
    st["lens"] = ints(total)
    r = random.Random(seed)

    def pages_for(need, spare=3):
        """Page ids of each row, all over a pool with a few pages to spare."""
        ids = list(range(sum(need) + spare))
        r.shuffle(ids)
        at, rows = 0, []
        for m in need:
            rows.append(ids[at:at + m])
            at += m
        return rows, len(ids)

    def padded(rows, fill):
        width = max(1, max(len(x) for x in rows))
        return ints([x + [fill] * (width - len(x)) for x in rows])

    def pool16(pages, size):
        shape = (pages, KV, size, D) if c["hnd"] else (pages, size, KV, D)
        return rand(*shape).transpose(1, 2) if c["hnd"] else rand(*shape)

    def pool8(pages):
        """Codes [page, position, kv head, dim] and their rows' scales: values of earlier conversations where nothing was written yet."""
        shape = (pages, KV, page, D) if c["hnd"] else (pages, page, KV, D)
        x = rand(*shape, dtype=torch.float32)
        d = x.abs().amax(-1, keepdim=True) / TOP
        x = (x / d).to(E4M3)
        d = d[..., 0]
        return (x.transpose(1, 2), d) if c["hnd"] else (x, d.transpose(1, 2))

    shared = c["op"] == "shared"
    own_pages = [-(-t // page) for t in total]
    if shared:  # a sequence's table names the prefix's whole pages first, then its own
        held = [plen[g] // page if g >= 0 else 0 for g in group]
        rows, count = pages_for([-(-p // page) for p in plen] + [max(0, m - h) for m, h in zip(own_pages, held)])
        firsts, own_rows = rows[:len(plen)], rows[len(plen):]
        e4m3 = c["cache"] == "e4m3"
        st["ptable"] = padded(firsts, 0)
        table = [(([-1] * h if e4m3 else firsts[g][:h]) + x)[:m] for x, g, h, m in zip(own_rows, group, held, own_pages)]
        st["table"] = padded(table, 0)
        st["plens"] = ints(plen)
        cu = [sum(1 for g in group if 0 <= g < k) for k in range(len(plen) + 1)]
        st["cu"] = ints(cu)
        st["group"] = torch.tensor([max(g, 0) for g in group], device=dev)
        st["plen"] = torch.tensor([plen[g] if g >= 0 else 0 for g in group], device=dev)
        st["pk"], st["pv"] = pool16(count, page), pool16(count, page)
    else:
        rows, count = pages_for(own_pages)
        st["table"] = padded(rows, 0)
    if not shared or c["cache"] == "e4m3":
        (st["k"], dk), (st["v"], dv) = pool8(count), pool8(count)
        st["scales"] = torch.stack([dk, dv], 2).contiguous()  # [page, kv head, k and v, position]
    else:
        st["k"], st["v"] = st["pk"], st["pv"]
    if c["op"] == "append8":
        H, it = c["heads"], DTYPE[c["inp"]]
        seq_of = [s for s, m in enumerate(new) for _ in range(m)]
        st["seq_of"] = torch.tensor(seq_of, dtype=torch.int64, device=dev)
        st["pos"] = torch.tensor([total[s] - m + i for s, m in enumerate(new) for i in range(m)], dtype=torch.int64, device=dev)
        cu = [0]
        for m in new:
            cu.append(cu[-1] + m)
        st["cu"] = ints(cu)
        if c["fused"]:  # rows of one projection
            qkv = rand(n, H + 2 * KV, D, dtype=it)
            st["q"], st["k_new"], st["v_new"] = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
        else:
            st["q"], st["k_new"], st["v_new"] = rand(n, H, D, dtype=it), rand(n, KV, D, dtype=it), rand(n, KV, D, dtype=it)
        st["q_norm"] = 1 + 0.1 * rand(D, dtype=torch.float32) if c["norm"] else None
        st["k_norm"] = 1 + 0.1 * rand(D, dtype=torch.float32) if c["norm"] else None
        st["rope"] = rope_table(max(total) + 1, D, dev) if c["rope"] else None
    elif c["op"] == "read8":
        rows, count = pages_for([-(-t // c["to_page"]) for t in total])
        st["to_table"], st["to_page"] = padded(rows, 0), c["to_page"]
        st["to_k"], st["to_v"] = pool16(count, c["to_page"]), pool16(count, c["to_page"])
    else:
        st["heads"], st["q"] = c["heads"], rand(n, c["heads"], D)
    if own:
        import rpgbarengine_b200 as rb
        st["cache"] = rb.PagedKV8(st["k"], st["v"], st["scales"], dtype=dt) if "scales" in st else rb.PagedKV(st["k"], st["v"])
        st["batch"] = rb.PagedBatch(st["table"], st["lens"], cu_q=st["cu"], n_tokens=n) if c["op"] == "append8" else \
            rb.PagedBatch(st["table"], st["lens"])
        if c["op"] == "read8":
            st["to"] = rb.PagedKV(st["to_k"], st["to_v"])
        if shared:
            first = st["cache"] if c["cache"] == "same" else rb.PagedKV(st["pk"], st["pv"])
            st["prefix"] = rb.PagedPrefix(first, st["ptable"], st["plens"], st["cu"])
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


def quant_plain(x):
    """Codes and scales of rows."""
    d = (x.abs().amax(-1) / TOP).clamp(min=2.0 ** -126)
    return (x / d[..., None]).to(E4M3), d


def values_plain(st, at, which):
    """Values in 32 bits of the cache's slots (page, slot) `at`: [.., kv head, dim]."""
    page, slot = at
    pool = (st["k"], st["v"])[which]
    if "scales" not in st:
        return pool[page, slot].float()
    codes = pool.view(torch.uint8)[page, slot].view(E4M3).float()
    return codes * st["scales"][:, :, which].transpose(1, 2)[page, slot][..., None]


def gather_plain(st, which):
    """[sequence, kv head, place, dim] of every sequence, in 32 bits."""
    t = torch.arange(st["max_len"], device="cuda")
    page = st["table"][:, (t // st["page"]).clamp(max=st["table"].shape[1] - 1)].long().clamp(min=0)
    x = values_plain(st, (page, (t % st["page"]).expand_as(page)), which)
    if st["op"] == "shared":
        rows = st["ptable"][st["group"]]
        page = rows[:, (t // st["page"]).clamp(max=rows.shape[1] - 1)].long()
        first = st[("pk", "pv")[which]][page, (t % st["page"]).expand_as(page)].float()
        x = torch.where((t < st["plen"][:, None])[..., None, None], first, x)
    return x.transpose(1, 2)


def attend_plain(st):
    k = gather_plain(st, 0)
    S, KV, L, D = k.shape
    q = st["q"].float().view(S, KV, -1, D)
    s = q @ k.transpose(-1, -2) * D ** -0.5
    del k
    seen = (torch.arange(L, device="cuda") < st["lens"][:, None])[:, None, None]
    s = s.masked_fill(~seen, float("-inf"))
    m = s.amax(-1, keepdim=True)
    e = (s - torch.where(m > float("-inf"), m, 0.0)).exp()
    p = e / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return (p @ gather_plain(st, 1)).view(S, -1, D).to(st["io"])


def append_plain(st):
    q = norm_rope_plain(st["q"], st["q_norm"], st["rope"], st["pos"]).to(st["io"])
    k, dk = quant_plain(norm_rope_plain(st["k_new"], st["k_norm"], st["rope"], st["pos"]))
    v, dv = quant_plain(st["v_new"].float())
    page, slot = st["table"][st["seq_of"], st["pos"] // st["page"]].long(), st["pos"] % st["page"]
    st["k"].view(torch.uint8)[page, slot] = k.view(torch.uint8)
    st["v"].view(torch.uint8)[page, slot] = v.view(torch.uint8)
    st["scales"][page, :, :, slot] = torch.stack([dk, dv], 2)
    return {"q": q, "k": st["k"], "v": st["v"], "scales": st["scales"]}


def read_plain(st):
    t = torch.arange(st["max_len"], device="cuda")
    seq, pos = (t < st["lens"][:, None]).nonzero(as_tuple=True)
    src = st["table"][seq, pos // st["page"]].long(), pos % st["page"]
    dst = st["to_table"][seq, pos // st["to_page"]].long(), pos % st["to_page"]
    st["to_k"][dst] = values_plain(st, src, 0).to(st["io"])
    st["to_v"][dst] = values_plain(st, src, 1).to(st["io"])
    return {"k": st["to_k"], "v": st["to_v"]}


def run(state):
    st = state
    if not own:
        return append_plain(st) if st["op"] == "append8" else read_plain(st) if st["op"] == "read8" else {"out": attend_plain(st)}
    import rpgbarengine_b200 as rb
    if st["op"] == "append8":
        q = rb.paged_append(st["cache"], st["batch"], st["q"], st["k_new"], st["v_new"], q_norm=st["q_norm"], k_norm=st["k_norm"],
                            eps=EPS, rope=st["rope"])
        return {"q": q, "k": st["k"], "v": st["v"], "scales": st["scales"]}
    if st["op"] == "read8":
        rb.paged_read(st["cache"], st["batch"], st["to"], st["to_table"])
        return {"k": st["to_k"], "v": st["to_v"]}
    if st["op"] == "shared":
        return {"out": rb.paged_attention_decode(st["cache"], st["batch"], st["q"], prefix=st["prefix"])}
    return {"out": rb.paged_attention_decode(st["cache"], st["batch"], st["q"])}


# --------------------------------------------------------------- 64 bits
def exact(case, seed):
    """From the definitions, a sequence at a time, in 64 bits; codes as they are before their rounding."""
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    new, total, plen, group = lengths(case)
    D, size = case["hd"], case["page"]

    def slots(row, count, size):
        p = torch.arange(count, device="cuda")
        return row.long()[p // size], p % size

    def held(s, count):
        """K and V [position, kv head, dim] of a sequence's own pages."""
        pg, sl = slots(st["table"][s], count, size)
        pg = pg.clamp(min=0)
        if "scales" not in st:
            return [x[pg, sl].double() for x in (st["k"], st["v"])]
        kv = [x.view(torch.uint8)[pg, sl].view(E4M3).double() for x in (st["k"], st["v"])]
        d = st["scales"][pg, :, :, sl].double()
        return [kv[0] * d[:, :, 0, None], kv[1] * d[:, :, 1, None]]

    if case["op"] == "append8":
        def turned(x, gain):
            x = x.double()
            if gain is not None:
                x = x / ((x * x).sum(-1, keepdim=True) / D + EPS).sqrt() * gain.double()
            if st["rope"] is None:
                return x
            cos, sin = st["rope"].double()[st["pos"]].chunk(2, -1)
            z = torch.complex(x[..., : D // 2], x[..., D // 2:]) * torch.complex(cos, sin)[:, None]
            return torch.cat([z.real, z.imag], -1)

        k, v, scales = st["k"].double(), st["v"].double(), st["scales"].double()
        for x, pool, w in ((turned(st["k_new"], st["k_norm"]), k, 0), (st["v_new"].double(), v, 1)):
            d = torch.maximum(x.abs().max(-1).values / TOP, torch.tensor(2.0 ** -126, dtype=torch.float64, device="cuda"))
            at = 0
            for s, m in enumerate(new):
                if m:
                    pg, sl = (y[total[s] - m:] for y in slots(st["table"][s], total[s], size))
                    pool[pg, sl] = x[at:at + m] / d[at:at + m, :, None]
                    scales[pg, :, w, sl] = d[at:at + m]
                at += m
        return {"q": turned(st["q"], st["q_norm"]), "k": k, "v": v, "scales": scales}
    if case["op"] == "read8":
        to = [st["to_k"].double(), st["to_v"].double()]
        for s, t in enumerate(total):
            if t:
                at = slots(st["to_table"][s], t, case["to_page"])
                for x, y in zip(to, held(s, t)):
                    x[at] = y
        return {"k": to[0], "v": to[1]}
    out = torch.zeros(st["n"], case["heads"], D, dtype=torch.float64, device="cuda")
    for s, t in enumerate(total):
        if t:
            k, v = held(s, t)
            if group[s] >= 0:
                p = min(t, plen[group[s]])
                at = slots(st["ptable"][group[s]], p, size)
                k, v = torch.cat([st["pk"][at].double(), k[p:]]), torch.cat([st["pv"][at].double(), v[p:]])
            q = st["q"][s].double().view(case["kv"], -1, D)
            a = torch.softmax(torch.einsum("kgd,tkd->kgt", q, k) / D ** 0.5, -1)
            out[s] = torch.einsum("kgt,tkd->kgd", a, v).reshape(-1, D)
    return {"out": out}
