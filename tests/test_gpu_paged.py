"""Paged-cache operators on the GPU against their definitions in 64 bits.

Tolerances: an attention output may differ from the exact value e = sum p v by
the rounding of the output to 16 bits, u |e|, and by the rounding of the
probabilities to 16 bits before their product with V, u sum p |v| (u = 2^-8
for bfloat16, 2^-11 for float16); a quarter of that again covers the fp32
scores, exponentials and sums, whose error is below 2^-13 of sum p |v|.
Append rounds once, after fp32 arithmetic within 2^-20 of the row's largest
value.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import rpgbarengine_b200 as rb  # noqa: E402
from rpgbarengine_b200 import paged  # noqa: E402

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
    if not torch.cuda.is_available() or rb.device_count() == 0:
        pytest.fail("GPU test collected without a CUDA device")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make_pool(g, lens, page, kv, hd, dtype, hnd=False, spare=3, width=0):
    """Pools full of values, with a table that spreads the sequences' pages
    over them; unused entries of a row name no page."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    shape = (pages, kv, page, hd) if hnd else (pages, page, kv, hd)
    k, v = randn(g, *shape, dtype=dtype), randn(g, *shape, dtype=dtype)
    if hnd:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    perm = torch.randperm(pages, generator=g, device="cuda").tolist()
    width = max(width, 1, max(need))
    table, at = [], 0
    for n in need:
        table.append(perm[at:at + n] + [-1] * (width - n))
        at += n
    return k, v, table


def rows_of(pool, table_row, n):
    """Positions [0, n) of a sequence: (values [n, kv, hd] in 64 bits, present [n])."""
    page = pool.shape[1]
    vals = torch.zeros(n, *pool.shape[2:], dtype=torch.float64, device="cuda")
    there = torch.zeros(n, dtype=torch.bool, device="cuda")
    for j, p in enumerate(table_row):
        a, b = j * page, min(n, (j + 1) * page)
        if a < n and 0 <= p < pool.shape[0]:
            vals[a:b] = pool[p, : b - a].double()
            there[a:b] = True
    return vals, there


def attend(q, k, v, there, first, scale):
    """(out, sum p |v|): q [m, H, d], row i at position first + i, over k, v [n, kv, d] in 64 bits."""
    m, H, d = q.shape
    n, kv = k.shape[0], k.shape[1]
    out = torch.zeros(m, H, d, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    if n == 0 or m == 0:
        return out, mag
    seen = (torch.arange(n, device="cuda") <= first + torch.arange(m, device="cuda")[:, None]) & there
    for h in range(H):
        s = q[:, h].double() @ k[:, h * kv // H].T * scale
        s = s.masked_fill(~seen, float("-inf"))
        top = s.amax(1, keepdim=True)
        e = torch.exp(s - torch.where(top.isinf(), 0.0, top))
        z = e.sum(1, keepdim=True)
        p = torch.where(z > 0, e / z, 0.0)
        out[:, h], mag[:, h] = p @ v[:, h * kv // H], p @ v[:, h * kv // H].abs()
    return out, mag


def close(got, want, mag):
    u = U[got.dtype]
    assert torch.isfinite(got).all()
    over = (got.double() - want).abs() - 1.25 * u * (want.abs() + mag)
    assert float(over.max()) <= 1e-30, (float(over.max()), int((over > 0).sum()))


# ------------------------------------------------------------------ append
def turned(x, gain, rope, pos, eps):
    x = x.double()
    if gain is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * gain.double()
    if rope is not None:
        h = x.shape[-1] // 2
        c, s = rope[pos, None, :h].double(), rope[pos, None, h:].double()
        x = torch.cat([x[..., :h] * c - x[..., h:] * s, x[..., h:] * c + x[..., :h] * s], -1)
    return x


APPEND = [  # new tokens, prefix, heads, kv, hd, page, cache, in, norm, rope, hnd, fused
    ([1], [0], 16, 8, 128, 16, "f16", "f32", True, True, False, False),
    ([1] * 7, [0, 5, 15, 16, 63, 64, 1000], 32, 8, 128, 64, "bf16", "f32", True, True, False, False),
    ([3, 0, 130, 1, 0], [0, 9, 62, 255, 0], 4, 2, 64, 16, "bf16", "bf16", True, True, True, True),
    ([200], [100], 5, 1, 128, 256, "f16", "f16", False, True, False, True),
    ([33, 40], [0, 1], 3, 3, 64, 32, "f16", "f32", True, False, True, True),
    ([64, 2], [0, 77], 16, 1, 128, 128, "bf16", "f32", False, False, False, False),
    ([1, 1, 1], [3, 4, 5], 12, 4, 64, 64, "bf16", "f16", True, True, False, False),
    ([1] * 70, list(range(70)), 8, 8, 128, 16, "bf16", "f32", True, True, False, True),
]


def append_inputs(g, n, H, kv, hd, ty, fused):
    dt = {"f32": torch.float32, **DT}[ty]
    if fused:
        x = randn(g, n, H + 2 * kv, hd, dtype=dt)
        return x[:, :H], x[:, H:H + kv], x[:, H + kv:]
    return tuple(randn(g, n, h, hd, dtype=dt) for h in (H, kv, kv))


@pytest.mark.parametrize("new,pre,H,kv,hd,page,cache,ty,norm,rope,hnd,fused", APPEND)
def test_append(new, pre, H, kv, hd, page, cache, ty, norm, rope, hnd, fused):
    g = gen(len(new) + H)
    dt = DT[cache]
    lens = [a + b for a, b in zip(new, pre)]
    k, v, table = make_pool(g, lens, page, kv, hd, dt, hnd)
    k0, v0, n = k.clone(), v.clone(), sum(new)
    q, kn, vn = append_inputs(g, n, H, kv, hd, ty, fused)
    qg, kg = (1 + 0.1 * randn(g, hd), 1 + 0.1 * randn(g, hd)) if norm else (None, None)
    tab = rb.rope_table(max(lens) + 1, hd) if rope else None
    single = all(m == 1 for m in new)
    cu = None if single else i32(np.concatenate([[0], np.cumsum(new)]).tolist())
    status = i32([0])
    batch = rb.PagedBatch(i32(table), i32(lens), cu, n, status)
    got = rb.paged_append(rb.PagedKV(k, v), batch, q, kn, vn, qg, kg, 1e-6, tab)
    pos = torch.tensor([b + i for a, b in zip(new, pre) for i in range(a)], device="cuda")
    seq = [s for s, a in enumerate(new) for _ in range(a)]
    u = U[dt]

    def near(a, want):
        assert bool(((a.double() - want).abs() <= u * want.abs() + 2.0 ** -20 * want.abs().amax(-1, keepdim=True) + 2.0 ** -25).all())

    near(got, turned(q, qg, tab, pos, 1e-6))
    wk, wv = turned(kn, kg, tab, pos, 1e-6), vn.double()
    touched = torch.zeros(k.shape[:2], dtype=torch.bool, device="cuda")
    for i, s in enumerate(seq):
        p = int(pos[i])
        pg, sl = table[s][p // page], p % page
        near(k[pg, sl], wk[i])
        near(v[pg, sl], wv[i])
        touched[pg, sl] = True
    assert torch.equal(k[~touched], k0[~touched]) and torch.equal(v[~touched], v0[~touched])
    assert int(status) == 0


def test_append_drops_tokens_without_a_place():
    g = gen(3)
    kv, hd, page, H = 2, 128, 16, 4
    k, v, _ = make_pool(g, [64], page, kv, hd, torch.bfloat16)
    k0, v0 = k.clone(), v.clone()
    # a page that is not there, an id past the pool, a position past the table,
    # one past the rope rows, fewer positions than new tokens, and one that fits
    table = [[-1, 0], [k.shape[0], 0], [0, 1], [0, 1], [2, 3], [1, 4]]
    lens = [10, 5, 33, 31, 1, 18]
    new = [1, 1, 1, 1, 2, 1]
    cu = i32(np.concatenate([[0], np.cumsum(new)]).tolist())
    q, kn, vn = append_inputs(g, 7, H, kv, hd, "f32", False)
    tab = rb.rope_table(30, hd)
    for use_status in (True, False):
        k.copy_(k0), v.copy_(v0)
        status = i32([0]) if use_status else None
        batch = rb.PagedBatch(i32(table), i32(lens), cu, 7, status)
        got = rb.paged_append(rb.PagedKV(k, v), batch, q, kn, vn, rope=tab)
        assert not use_status or int(status) == paged.DROPPED
        assert bool((got[:5] == 0).all()) and bool((got[5:] != 0).any(-1).all())
        changed = (k != k0).any(-1).any(-1).nonzero().tolist()
        assert changed == [[2, 0], [4, 1]], changed


# Enough tokens that a warp takes several heads: counts that leave the last warp
# and its last step part full, q, k and v rows in one step, pages that are not there.
MANY = [  # heads, kv, hd, in, fused
    (5, 1, 64, "f16", True),
    (5, 1, 128, "f32", False),
    (7, 7, 128, "bf16", False),
    (12, 4, 64, "f32", True),
    (32, 8, 128, "f16", True),
    (9, 3, 64, "bf16", True),
    (1, 1, 128, "f16", False),
]


@pytest.mark.parametrize("H,kv,hd,ty,fused", MANY)
def test_append_of_many_tokens(H, kv, hd, ty, fused):
    g = gen(H + hd)
    new, pre, page, dt = [2500, 0, 1, 3100, 777], [17, 5, 0, 300, 64], 32, torch.bfloat16 if ty == "bf16" else torch.float16
    lens, n = [a + b for a, b in zip(new, pre)], sum(new)
    k, v, table = make_pool(g, lens, page, kv, hd, dt)
    table[0][3], table[3][100] = -1, k.shape[0]  # the pages of 64 new tokens
    k0, v0 = k.clone(), v.clone()
    q, kn, vn = append_inputs(g, n, H, kv, hd, ty, fused)
    qg, kg, tab = 1 + 0.1 * randn(g, hd), 1 + 0.1 * randn(g, hd), rb.rope_table(max(lens), hd)
    cu, status = i32(np.concatenate([[0], np.cumsum(new)]).tolist()), i32([0])
    got = rb.paged_append(rb.PagedKV(k, v), rb.PagedBatch(i32(table), i32(lens), cu, n, status), q, kn, vn, qg, kg, 1e-6, tab)
    pos = torch.tensor([b + i for a, b in zip(new, pre) for i in range(a)], device="cuda")
    seq = torch.tensor([s for s, a in enumerate(new) for _ in range(a)], device="cuda")
    pages = i32(table)[seq, pos // page].long()
    there = (pages >= 0) & (pages < k.shape[0])
    assert int((~there).sum()) == 64 and int(status) == paged.DROPPED
    assert bool((got[~there] == 0).all())
    u, pg, sl = U[dt], pages[there], pos[there] % page

    def near(a, want):
        assert bool(((a.double() - want).abs() <= u * want.abs() + 2.0 ** -20 * want.abs().amax(-1, keepdim=True) + 2.0 ** -25).all())

    near(got[there], turned(q, qg, tab, pos, 1e-6)[there])
    near(k[pg, sl], turned(kn, kg, tab, pos, 1e-6)[there])
    near(v[pg, sl], vn.double()[there])
    touched = torch.zeros(k.shape[:2], dtype=torch.bool, device="cuda")
    touched[pg, sl] = True
    assert torch.equal(k[~touched], k0[~touched]) and torch.equal(v[~touched], v0[~touched])


# ------------------------------------------------------------------ decode
DECODE = [  # lens, heads, kv, hd, page, cache, hnd
    ([1], 16, 8, 128, 16, "f16", False),
    ([33], 16, 8, 128, 16, "bf16", False),
    ([0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 0], 32, 8, 128, 64, "bf16", False),
    ([0, 0, 0], 4, 2, 64, 32, "f16", True),
    ([4200], 32, 8, 128, 64, "bf16", False),
    ([4097, 3], 16, 1, 128, 256, "f16", False),
    ([700, 1, 90, 0, 513], 5, 1, 128, 128, "bf16", True),
    ([1000, 999, 77], 12, 4, 64, 16, "f16", False),
    ([257, 511, 1024, 8], 12, 12, 64, 32, "bf16", True),
    ([1100 + 7 * i for i in range(24)], 32, 4, 128, 64, "f16", False),
    ([(37 * i) % 400 for i in range(200)], 8, 8, 128, 16, "bf16", False),
    ([20000], 3, 3, 64, 128, "bf16", False),
    ([640, 5000, 1], 14, 2, 128, 32, "f16", True),
]


def decode_case(lens, H, kv, hd, page, cache, hnd, seed=0, spread=1.0):
    g = gen(seed + len(lens) + hd)
    dt = DT[cache]
    k, v, table = make_pool(g, lens, page, kv, hd, dt, hnd)
    q = (randn(g, len(lens), H, hd) * spread).to(dt)
    return k, v, table, q


def check_decode(got, q, k, v, table, lens, scale):
    reach = len(table[0]) * k.shape[1]
    for s, n in enumerate(lens):
        m = min(n, reach)
        kk, there = rows_of(k, table[s], m)
        vv, _ = rows_of(v, table[s], m)
        want, mag = attend(q[s:s + 1], kk, vv, there, n - 1, scale)
        close(got[s:s + 1], want, mag)


@pytest.mark.parametrize("lens,H,kv,hd,page,cache,hnd", DECODE)
def test_decode(lens, H, kv, hd, page, cache, hnd):
    k, v, table, q = decode_case(lens, H, kv, hd, page, cache, hnd)
    got = rb.paged_attention_decode(rb.PagedKV(k, v), rb.PagedBatch(i32(table), i32(lens)), q)
    check_decode(got, q, k, v, table, lens, hd ** -0.5)


@pytest.mark.parametrize("cache", ["bf16", "f16"])
@pytest.mark.parametrize("spread,scale", [(8.0, 0.3), (0.01, 0.0884), (1.0, 1e-3)])
def test_decode_peaked_and_flat(cache, spread, scale):
    lens = [3000, 40, 513]
    k, v, table, q = decode_case(lens, 16, 4, 128, 64, cache, False, 5, spread)
    got = rb.paged_attention_decode(rb.PagedKV(k, v), rb.PagedBatch(i32(table), i32(lens)), q, scale=scale)
    check_decode(got, q, k, v, table, lens, float(np.float32(scale)))


def test_decode_missing_pages_and_unused_values():
    # pages given back (-1), ids past the pool, a length past the table; NaN
    # and infinities in every slot that no sequence holds
    page, kv, H, hd = 16, 2, 8, 128
    lens = [200, 130, 7, 90, 64]
    k, v, table, q = decode_case(lens, H, kv, hd, page, "bf16", False, 9)
    table[0][0] = table[0][1] = -1
    table[0][7] = 10 ** 6
    table[1][8] = -5  # the page of its last positions
    table[2][0] = -1  # nothing left to see
    lens[3] = 10 ** 6  # past the table: its row's unnamed pages are not there
    used = torch.zeros(k.shape[:2], dtype=torch.bool, device="cuda")
    for s, n in enumerate(lens):
        for j, p in enumerate(table[s]):
            if 0 <= p < k.shape[0]:
                used[p, : max(0, min(page, n - j * page))] = True
    for bad in (float("nan"), float("inf"), float("-inf")):
        k[~used], v[~used] = bad, bad
        got = rb.paged_attention_decode(rb.PagedKV(k, v), rb.PagedBatch(i32(table), i32(lens)), q)
        check_decode(got, q, k, v, table, lens, hd ** -0.5)
        assert bool((got[2] == 0).all())


def test_decode_shared_pages_and_strided_q():
    # two sequences on the same prefix pages; q a slice of a wider projection
    page, kv, H, hd = 64, 4, 12, 64
    k, v, table, _ = decode_case([300, 300], H, kv, hd, page, "f16", True, 2)
    table[1][:3] = table[0][:3]
    wide = randn(gen(4), 2, H + 2 * kv, hd, dtype=torch.float16)
    q = wide[:, 4:4 + H]
    got = rb.paged_attention_decode(rb.PagedKV(k, v), rb.PagedBatch(i32(table), i32([300, 260])), q)
    check_decode(got, q, k, v, table, [300, 260], hd ** -0.5)


def test_decode_lengths_change_between_calls_and_in_a_graph():
    # one batch, its lengths updated in place: every call starts afresh, the
    # same answer for the same lengths bit for bit, and a captured call follows
    page, kv, H, hd = 32, 8, 32, 128
    most = [900, 1500, 40, 8, 2000]
    k, v, table, q = decode_case(most, H, kv, hd, page, "bf16", False, 1)
    lens = i32([0] * 5)
    cache, batch = rb.PagedKV(k, v), rb.PagedBatch(i32(table), lens)
    out = torch.empty_like(q)
    rb.paged_attention_decode(cache, batch, q, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rb.paged_attention_decode(cache, batch, q, out=out)
    for cur in ([900, 1500, 40, 8, 2000], [1, 0, 40, 7, 1999], [899, 1, 0, 0, 0], [900, 1500, 40, 8, 2000]):
        lens.copy_(i32(cur))
        a = rb.paged_attention_decode(cache, batch, q)
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        check_decode(a, q, k, v, table, cur, hd ** -0.5)
        assert torch.equal(a, out)


def test_many_sequences():
    # more sequences than a warp's lanes many times over, most of them empty or
    # of one position, in decode and as prompts of one and of a few tokens
    page, kv, H, hd = 16, 2, 4, 64
    lens = [0 if i % 3 == 0 else 1 if i % 7 else (i * 37) % 90 for i in range(3001)]
    k, v, table, q = decode_case(lens, H, kv, hd, page, "f16", False, 4)
    cache = rb.PagedKV(k, v)
    tab, ln = i32(table), i32(lens)
    kk, vv = (x.double()[tab.clamp(min=0).long()].flatten(1, 2) for x in (k, v))  # [sequence, place, head, dim]

    def want(qs, seq, last):
        s = torch.einsum("nhgd,nthd->nhgt", qs.double().view(len(seq), kv, H // kv, hd), kk[seq]) * hd ** -0.5
        far = torch.arange(kk.shape[1], device="cuda") > last[:, None]
        p = torch.where(far[:, None, None], 0.0, torch.exp(s))
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        f = lambda x: torch.einsum("nhgt,nthd->nhgd", p, x[seq]).reshape(len(seq), H, hd)  # noqa: E731
        return f(vv), f(vv.abs())

    seq = torch.arange(len(lens), device="cuda")
    close(rb.paged_attention_decode(cache, rb.PagedBatch(tab, ln), q), *want(q, seq, ln.long() - 1))
    close(rb.paged_attention_prompt(cache, rb.PagedBatch(tab, ln), q), *want(q, seq, ln.long() - 1))
    new = [min(n, 5) for n in lens]
    cu = i32(np.concatenate([[0], np.cumsum(new)]).tolist())
    n = sum(new)
    qp = randn(gen(1), n, H, hd, dtype=torch.float16)
    seq = torch.repeat_interleave(seq, torch.tensor(new, device="cuda"))
    last = ln.long()[seq] - cu.long()[seq + 1] + torch.arange(n, device="cuda")
    close(rb.paged_attention_prompt(cache, rb.PagedBatch(tab, ln, cu, n), qp), *want(qp, seq, last))


def test_decode_offsets_past_32_bits():
    # a pool of more than 2^31 values whose last pages hold the sequence
    page, kv, H, hd = 256, 8, 16, 128
    pages = (1 << 31) // (page * kv * hd) + 5
    cache = rb.PagedKV.empty(pages, page, kv, hd)
    g = gen(8)
    n = 1000
    table = [[pages - 1, pages - 3, 0, pages - 2]]
    for p in table[0]:
        cache.k[p] = randn(g, page, kv, hd, dtype=torch.bfloat16)
        cache.v[p] = randn(g, page, kv, hd, dtype=torch.bfloat16)
    q = randn(g, 1, H, hd, dtype=torch.bfloat16)
    got = rb.paged_attention_decode(cache, rb.PagedBatch(i32(table), i32([n])), q)
    check_decode(got, q, cache.k, cache.v, table, [n], hd ** -0.5)
    gp = rb.paged_attention_prompt(cache, rb.PagedBatch(i32(table), i32([n]), i32([0, 1]), 1), q)
    check_decode(gp, q, cache.k, cache.v, table, [n], hd ** -0.5)


# ------------------------------------------------------------------ prompts
PACKED = [  # lens, heads, kv, hd, type, fused
    ([1], 16, 8, 128, "f16", False),
    ([33], 16, 8, 128, "bf16", False),
    ([0, 1, 127, 0, 128, 129, 2, 64], 8, 2, 128, "bf16", True),
    ([512], 32, 8, 128, "bf16", True),
    ([700, 3, 255], 8, 8, 128, "f16", False),
    ([300, 41], 5, 1, 128, "bf16", True),
    ([200, 1000], 16, 1, 64, "f16", False),
    ([257, 0, 65], 12, 12, 64, "bf16", True),
    ([385, 130], 12, 4, 64, "f16", True),
    ([1, 1, 1, 1, 0, 1], 14, 2, 128, "bf16", False),
    ([2100], 4, 1, 128, "f16", False),
    ([31 * i % 90 for i in range(80)], 6, 2, 64, "bf16", False),
]


def packed_inputs(g, n, H, kv, hd, dt, fused):
    if fused:
        x = randn(g, n, H + 2 * kv, hd, dtype=dt)
        return x[:, :H], x[:, H:H + kv], x[:, H + kv:]
    return tuple(randn(g, n, h, hd, dtype=dt) for h in (H, kv, kv))


def check_packed(got, q, k, v, lens, scale):
    at = 0
    for n in lens:
        kk, vv = k[at:at + n].double(), v[at:at + n].double()
        want, mag = attend(q[at:at + n], kk, vv, torch.ones(n, dtype=torch.bool, device="cuda"), 0, scale)
        if n:
            close(got[at:at + n], want, mag)
        at += n


@pytest.mark.parametrize("lens,H,kv,hd,ty,fused", PACKED)
def test_packed_prompt(lens, H, kv, hd, ty, fused):
    g = gen(len(lens) + hd + H)
    n = sum(lens)
    q, k, v = packed_inputs(g, n, H, kv, hd, DT[ty], fused)
    cu = i32(np.concatenate([[0], np.cumsum(lens)]).tolist())
    status = i32([0])
    got = rb.attention_prompt(q, k, v, cu, status=status)
    check_packed(got, q, k, v, lens, hd ** -0.5)
    assert int(status) == 0


@pytest.mark.parametrize("ty", ["bf16", "f16"])
@pytest.mark.parametrize("spread,scale", [(6.0, 0.3), (0.01, 0.0884), (1.0, 1e-3)])
def test_packed_prompt_peaked_and_flat(ty, spread, scale):
    g = gen(12)
    lens = [600, 90]
    q, k, v = packed_inputs(g, 690, 8, 2, 128, DT[ty], False)
    q = (q.float() * spread).to(q.dtype)
    got = rb.attention_prompt(q, k, v, i32([0, 600, 690]), scale=scale)
    check_packed(got, q, k, v, lens, float(np.float32(scale)))


def test_packed_prompt_growing_scores():
    # keys whose scores rise along the sequence: the running maximum moves at
    # every step, so every partial sum is rescaled again and again
    for ty in ("bf16", "f16"):
        n, H, kv, hd = 1000, 4, 2, 128
        g = gen(3)
        q = torch.ones(n, H, hd, device="cuda", dtype=DT[ty])
        ramp = torch.linspace(-40, 40, n, device="cuda")[:, None, None]
        k = (ramp + 0.01 * randn(g, n, kv, hd)).to(DT[ty])
        v = randn(g, n, kv, hd, dtype=DT[ty])
        got = rb.attention_prompt(q, k, v, i32([0, n]), scale=0.02)
        check_packed(got, q, k, v, [n], float(np.float32(0.02)))


@pytest.mark.parametrize("H,kv", [(6, 2), (5, 1), (12, 12), (14, 2), (16, 2)])
@pytest.mark.parametrize("ty", ["bf16", "f16"])
def test_packed_prompt_repeats_bit_for_bit(H, kv, ty):
    # rows of a tile that belong to no token hold what an earlier call left
    # there: whatever that was, the tokens' rows come out the same
    g = gen(H)
    lens = [900, 77, 300]
    q, k, v = packed_inputs(g, sum(lens), H, kv, 128, DT[ty], False)
    cu = i32([0, 900, 977, 1277])
    want = rb.attention_prompt(q, k, v, cu)
    for scale in (1e3, 1e-3, float("inf")):
        junk = (randn(g, 2000, 8, 128) * scale).to(DT[ty])
        rb.attention_prompt(junk, junk, junk, i32([0, 2000]))
        assert torch.equal(rb.attention_prompt(q, k, v, cu), want)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_packed_prompt_later_positions_do_not_leak(bad):
    # what a row may not see cannot change it, whatever it holds: the key and
    # the value at position 300, and the whole sequence that follows
    g = gen(21)
    H, kv, hd = 8, 2, 128
    q, k, v = packed_inputs(g, 500, H, kv, hd, torch.bfloat16, False)
    cu = i32([0, 430, 500])
    want = rb.attention_prompt(q, k, v, cu)
    k2, v2 = k.clone(), v.clone()
    k2[300], v2[300] = bad, bad
    k2[430:], v2[430:] = bad, bad
    got = rb.attention_prompt(q, k2, v2, cu)
    check_packed(got[:300], q[:300], k[:300], v[:300], [300], hd ** -0.5)
    assert torch.isfinite(want).all()
    assert torch.isnan(got[300:430]).all()  # these see it (infinite keys give scores of both signs at once)
    q2 = q.clone()
    q2[77], q2[78, 3] = bad, bad
    got = rb.attention_prompt(q2, k, v, cu)
    ok = torch.ones(500, H, dtype=torch.bool, device="cuda")
    ok[77], ok[78, 3] = False, False
    assert torch.isnan(got[~ok]).all() and torch.equal(got[ok], want[ok])


def test_prompt_rows_outside_every_sequence_are_left_alone():
    g = gen(2)
    q, k, v = packed_inputs(g, 300, 4, 2, 64, torch.float16, False)
    out = torch.full_like(q, 3.0)
    rb.attention_prompt(q, k, v, i32([10, 50, 260]), out=out)
    assert bool((out[:10] == 3).all()) and bool((out[260:] == 3).all())
    check_packed(out[10:260], q[10:260], k[10:260], v[10:260], [40, 210], 64 ** -0.5)
    # bounds that leave [0, n_tokens] or fall are kept inside it
    rb.attention_prompt(q, k, v, i32([-5, 100, 40, 9999]), out=out)
    torch.cuda.synchronize()


PAGED = [  # new, prefix, heads, kv, hd, page, cache, hnd
    ([1], [0], 16, 8, 128, 16, "f16", False),
    ([40, 1, 0, 7], [0, 300, 20, 1], 32, 8, 128, 64, "bf16", False),
    ([129, 64, 300], [256, 0, 100], 8, 2, 128, 16, "f16", True),
    ([500], [700], 16, 4, 64, 128, "bf16", False),
    ([3, 260], [1000, 5], 5, 1, 128, 256, "bf16", True),
    ([100, 90, 80], [31, 32, 33], 12, 12, 64, 32, "f16", True),
    ([1] * 9, [0, 1, 15, 16, 17, 127, 128, 129, 600], 16, 1, 64, 16, "bf16", False),
    ([768], [256], 8, 8, 128, 32, "bf16", False),
]


def check_paged(got, q, k, v, table, new, lens, scale):
    at, reach = 0, len(table[0]) * k.shape[1]
    for s, (m, n) in enumerate(zip(new, lens)):
        c = max(0, min(n, reach))
        kk, there = rows_of(k, table[s], c)
        vv, _ = rows_of(v, table[s], c)
        want, mag = attend(q[at:at + m], kk, vv, there, n - m, scale)
        if m:
            close(got[at:at + m], want, mag)
        at += m


@pytest.mark.parametrize("new,pre,H,kv,hd,page,cache,hnd", PAGED)
def test_paged_prompt(new, pre, H, kv, hd, page, cache, hnd):
    g = gen(len(new) + H + hd)
    lens = [a + b for a, b in zip(new, pre)]
    k, v, table = make_pool(g, lens, page, kv, hd, DT[cache], hnd)
    q = randn(g, sum(new), H, hd, dtype=DT[cache])
    cu = i32(np.concatenate([[0], np.cumsum(new)]).tolist())
    status = i32([0])
    got = rb.paged_attention_prompt(rb.PagedKV(k, v), rb.PagedBatch(i32(table), i32(lens), cu, sum(new), status), q)
    check_paged(got, q, k, v, table, new, lens, hd ** -0.5)
    assert int(status) == 0


def test_paged_prompt_missing_pages_short_caches_and_unused_values():
    page, kv, H, hd = 16, 2, 4, 128
    new, lens = [60, 50, 20, 300], [200, 30, 20, 300]  # the second holds fewer positions than new rows
    g = gen(5)
    k, v, table = make_pool(g, [200, 30, 20, 300], page, kv, hd, torch.bfloat16)
    table[0][2] = -1
    table[0][11] = 10 ** 7
    table[2][0] = table[2][1] = -1  # sees nothing at all
    table[3][0] = -1
    lens[3] = 310  # ten positions past its pages
    used = torch.zeros(k.shape[:2], dtype=torch.bool, device="cuda")
    for s, n in enumerate(lens):
        for j, p in enumerate(table[s]):
            if 0 <= p < k.shape[0]:
                used[p, : max(0, min(page, n - j * page))] = True
    q = randn(g, sum(new), H, hd, dtype=torch.bfloat16)
    cu = i32(np.concatenate([[0], np.cumsum(new)]).tolist())
    for bad in (float("nan"), float("inf")):
        k[~used], v[~used] = bad, bad
        got = rb.paged_attention_prompt(rb.PagedKV(k, v), rb.PagedBatch(i32(table), i32(lens), cu, sum(new)), q)
        check_paged(got, q, k, v, table, new, lens, hd ** -0.5)
        assert bool((got[110:130] == 0).all())


def test_one_token_each_through_the_prompt_call_agrees_with_decode():
    lens = [5, 129, 700]
    k, v, table, q = decode_case(lens, 16, 4, 128, 64, "bf16", False)
    cache, batch = rb.PagedKV(k, v), rb.PagedBatch(i32(table), i32(lens))
    check_decode(rb.paged_attention_prompt(cache, batch, q), q, k, v, table, lens, 128 ** -0.5)


# ---------------------------------------------------------- other layouts
@pytest.mark.parametrize("hd", [64, 128])
def test_pools_in_one_tensor_strided_rows_and_outputs_off_a_sector(hd):
    # K and V interleaved in one pool with room between heads, every second head
    # of a wider q, results on a 16-byte boundary that is no 32-byte one
    g = gen(hd)
    page, kv, H, pages = 32, 3, 6, 40
    pool = randn(g, pages, page, 2, kv + 1, 2 * hd, dtype=torch.bfloat16)
    before = pool.clone()
    k, v = pool[:, :, 0, :kv, :hd], pool[:, :, 1, 1:, hd:]
    lens, new = [300, 33, 130], [130, 1, 64]
    perm = torch.randperm(pages, generator=g, device="cuda").tolist()
    table = [perm[:10], perm[10:12] + [-1] * 8, perm[12:17] + [-1] * 5]
    n = sum(new)
    cu = i32(np.concatenate([[0], np.cumsum(new)]).tolist())
    wide = randn(g, n, 2 * H + 1, hd, dtype=torch.bfloat16)
    q = wide[:, 1::2]
    cache, batch = rb.PagedKV(k, v), rb.PagedBatch(i32(table), i32(lens), cu, n)

    def odd(shape):
        size = int(np.prod(shape))
        buf = torch.full((size + 16,), 5.0, dtype=torch.bfloat16, device="cuda")
        assert buf.data_ptr() % 32 == 0
        return buf, buf[8:8 + size].view(shape)

    buf, out = odd(q.shape)
    got = rb.paged_attention_prompt(cache, batch, q, out=out)
    assert got.data_ptr() == out.data_ptr()
    check_paged(out, q, k, v, table, new, lens, hd ** -0.5)
    assert bool((buf[:8] == 5).all()) and bool((buf[-8:] == 5).all())
    qd = q[:3]
    buf, out = odd(qd.shape)
    rb.paged_attention_decode(cache, rb.PagedBatch(i32(table), i32(lens)), qd, out=out)
    check_decode(out, qd, k, v, table, lens, hd ** -0.5)
    assert bool((buf[:8] == 5).all()) and bool((buf[-8:] == 5).all())
    buf, out = odd(q.shape)
    kk, vv = randn(g, n, 2 * kv, hd, dtype=torch.bfloat16)[:, ::2], randn(g, n, kv, 2 * hd, dtype=torch.bfloat16)[..., hd:]
    rb.attention_prompt(q, kk, vv, cu, out=out)
    check_packed(out, q, kk, vv, new, hd ** -0.5)
    assert bool((buf[:8] == 5).all()) and bool((buf[-8:] == 5).all())
    assert torch.equal(pool, before)
    # append into the same pool touches the new tokens' slots alone
    q_out = rb.paged_append(cache, batch, q, kk, vv)
    assert torch.equal(q_out, q)
    touched = torch.zeros_like(pool, dtype=torch.bool)
    at = 0
    for s, m in enumerate(new):
        for i in range(m):
            p = lens[s] - m + i
            pg, sl = table[s][p // page], p % page
            assert torch.equal(k[pg, sl], kk[at]) and torch.equal(v[pg, sl], vv[at])
            touched[pg, sl, 0, :kv, :hd] = True
            touched[pg, sl, 1, 1:, hd:] = True
            at += 1
    assert torch.equal(pool[~touched], before[~touched])


# ------------------------------------------------------ streams, refusals
def test_calls_on_another_stream():
    g = gen(6)
    q, k, v = packed_inputs(g, 400, 8, 2, 128, torch.bfloat16, False)
    cu = i32([0, 150, 400])
    want = rb.attention_prompt(q, k, v, cu)
    lens = [150, 250]
    kp, vp, table, qd = decode_case(lens, 8, 2, 128, 32, "bf16", False)
    cache, batch = rb.PagedKV(kp, vp), rb.PagedBatch(i32(table), i32(lens))
    wd = rb.paged_attention_decode(cache, batch, qd)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(20):
        got = rb.attention_prompt(q, k, v, cu, stream=side.cuda_stream)
        gd = rb.paged_attention_decode(cache, batch, qd, stream=side.cuda_stream)
        side.synchronize()
        assert torch.equal(got, want) and torch.equal(gd, wd)
        with torch.cuda.stream(side):
            got = rb.attention_prompt(q, k, v, cu)
        side.synchronize()
        assert torch.equal(got, want)


def test_wrapper_refusals():
    cache = rb.PagedKV.empty(4, 16, 2, 128)
    batch = rb.PagedBatch(i32([[0, 1]]), i32([5]))
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16, device="cuda")

    def refused(f):
        with pytest.raises(rb.RpgcError) as e:
            f()
        assert e.value.code == rb.E_ARG

    refused(lambda: rb.paged_attention_decode(cache, batch, q.half()))
    refused(lambda: rb.paged_attention_decode(cache, batch, q.cpu()))
    refused(lambda: rb.paged_attention_decode(cache, batch, torch.zeros(2, 4, 128, dtype=torch.bfloat16, device="cuda")))
    refused(lambda: rb.paged_attention_decode(cache, batch, torch.zeros(1, 3, 128, dtype=torch.bfloat16, device="cuda")))
    refused(lambda: rb.paged_attention_decode(cache, batch, q, scale=float("nan")))
    refused(lambda: rb.paged_attention_decode(cache, batch, q, scale=0.0))
    refused(lambda: rb.paged_attention_decode(cache, batch, q, out=torch.zeros_like(q).float()))
    refused(lambda: rb.paged_attention_decode(cache, rb.PagedBatch(i32([[0, 1]]), i32([5]), i32([0, 1]), 1), q))
    refused(lambda: rb.PagedBatch(i32([[0, 1]]).long(), i32([5])))
    refused(lambda: rb.PagedBatch(i32([[0, 1]]), i32([5, 6])))
    refused(lambda: rb.PagedBatch(i32([[0, 1]]), i32([5]), i32([0, 1])))
    refused(lambda: rb.PagedKV(cache.k, cache.v.half()))
    refused(lambda: rb.PagedKV(cache.k.float(), cache.v.float()))
    k = torch.zeros(1, 2, 128, device="cuda")
    refused(lambda: rb.paged_append(cache, batch, None, k, k.half()))
    refused(lambda: rb.paged_append(cache, batch, k, k, k, q_norm=torch.ones(128, device="cuda")))
    refused(lambda: rb.paged_append(cache, batch, None, k, k, rope=torch.zeros(4, 64, device="cuda")))
    odd = torch.zeros(1, 2, 132, device="cuda", dtype=torch.bfloat16)[..., 2:130]  # rows off a 16-byte boundary
    refused(lambda: rb.paged_append(cache, batch, None, odd, odd))
    refused(lambda: rb.attention_prompt(q, q, q, i32([0, 1]).long()))
    refused(lambda: rb.attention_prompt(q, q.half(), q.half(), i32([0, 1])))
    z = torch.zeros(1, 4, 96, dtype=torch.bfloat16, device="cuda")
    refused(lambda: rb.attention_prompt(z, z, z, i32([0, 1])))
    assert rb.paged_append(cache, batch, None, k, k) is None  # k and v alone are fine
    e = torch.zeros(0, 4, 128, dtype=torch.bfloat16, device="cuda")
    assert rb.attention_prompt(e, e, e, i32([0])).shape == (0, 4, 128)
