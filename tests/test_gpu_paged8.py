"""The 8-bit paged cache and shared prefixes on the GPU against their definitions in 64 bits.

Tolerances.  Attention: as in test_gpu_paged.py, the output's rounding u |e| and that of
the probabilities, u sum p |v|, a quarter of both for the fp32 arithmetic (u = 2^-8 for
bfloat16, 2^-11 for float16); codes and scales are the inputs, so their own rounding has no
part in it.  Append: fp32 arithmetic within 2^-20 of the row's largest value and as much in
the scale, so x / d is within 448 * 2^-19 of the exact quotient before it is rounded; half a
step of e4m3 is 2^-4 of the value, 2^-10 below 2^-6.  Reading back multiplies two fp32 values
and rounds: the same bits as in torch.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import rpgbarengine_b200 as rb  # noqa: E402
from rpgbarengine_b200 import paged  # noqa: E402

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E4M3 = torch.float8_e4m3fn


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


def ids_of(g, need, spare=3):
    """Rows of page ids, spread over a pool of that many pages and some more."""
    pages = sum(need) + spare
    perm = torch.randperm(pages, generator=g, device="cuda").tolist()
    rows, at = [], 0
    for n in need:
        rows.append(perm[at:at + n])
        at += n
    return rows, pages


def padded(rows, fill=-1, width=1):
    width = max([width] + [len(r) for r in rows])
    return [r + [fill] * (width - len(r)) for r in rows]


def pool16(g, pages, page, kv, hd, dtype, hnd=False):
    x = [randn(g, *((pages, kv, page, hd) if hnd else (pages, page, kv, hd)), dtype=dtype) for _ in range(2)]
    return [t.transpose(1, 2) for t in x] if hnd else x


def pool8(g, pages, page, kv, hd, hnd=False):
    """Codes and scales of random rows of different magnitudes."""
    out, sc = [], []
    for _ in range(2):
        x = randn(g, *((pages, kv, page, hd) if hnd else (pages, page, kv, hd)))
        d = x.abs().amax(-1, keepdim=True) / 448
        c = (x / d).to(E4M3)
        d = d[..., 0] * torch.exp2(torch.randint(-3, 3, d.shape[:-1], generator=g, device="cuda").float())
        out.append(c.transpose(1, 2) if hnd else c)
        sc.append(d if hnd else d.transpose(1, 2))
    return out[0], out[1], torch.stack(sc, 2).contiguous()


def values(cache, which):
    """[page, position, kv head, dim] in 64 bits."""
    pool = cache.k if which == 0 else cache.v
    if isinstance(cache, rb.PagedKV8):
        return pool.double() * cache.scales[:, :, which].transpose(1, 2).double()[..., None]
    return pool.double()


def rows_of(pool, table_row, a, b):
    """Positions [a, b) through a row of a table: values and which are there."""
    page = pool.shape[1]
    vals = torch.zeros(max(0, b - a), *pool.shape[2:], dtype=torch.float64, device="cuda")
    there = torch.zeros(max(0, b - a), dtype=torch.bool, device="cuda")
    for t in range(a, b):
        j = t // page
        p = table_row[j] if j < len(table_row) else -1
        if 0 <= p < pool.shape[0]:
            vals[t - a] = pool[p, t % page]
            there[t - a] = True
    return vals, there


def attend(q, k, v, there, scale):
    """(out, sum p |v|) of q [H, d] over k, v [n, kv, d] in 64 bits."""
    H, d = q.shape
    kv = k.shape[1]
    if not bool(there.any()):
        z = torch.zeros(H, d, dtype=torch.float64, device="cuda")
        return z, z
    s = torch.einsum("kgd,tkd->kgt", q.double().view(kv, -1, d), k) * scale
    p = torch.softmax(s.masked_fill(~there, float("-inf")), -1)
    return torch.einsum("kgt,tkd->kgd", p, v).reshape(H, d), torch.einsum("kgt,tkd->kgd", p, v.abs()).reshape(H, d)


def definition(cache, table, lens, q, scale, prefix=None):
    """prefix: (cache, table, plens, cu)."""
    K, V = values(cache, 0), values(cache, 1)
    if prefix:
        PK, PV = values(prefix[0], 0), values(prefix[0], 1)
    out, mag = [], []
    for s, n in enumerate(lens):
        n, own = max(0, n), 0
        k = v = there = None
        for g in range(len(prefix[2]) if prefix else 0):
            if prefix[3][g] <= s < prefix[3][g + 1]:
                own = min(n, max(0, prefix[2][g]))
                k, there = rows_of(PK, prefix[1][g], 0, own)
                v, _ = rows_of(PV, prefix[1][g], 0, own)
        k2, there2 = rows_of(K, table[s], own, n)
        v2, _ = rows_of(V, table[s], own, n)
        if k is not None:
            k2, v2, there2 = torch.cat([k, k2]), torch.cat([v, v2]), torch.cat([there, there2])
        o, m = attend(q[s], k2, v2, there2, scale)
        out.append(o)
        mag.append(m)
    return torch.stack(out), torch.stack(mag)


def close(got, want, mag):
    u = U[got.dtype]
    assert torch.isfinite(got).all()
    over = (got.double() - want).abs() - 1.25 * u * (want.abs() + mag)
    assert float(over.max()) <= 1e-30, (float(over.max()), int((over > 0).sum()), np.unravel_index(int(over.argmax()), over.shape))


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


APPEND = [  # new tokens, prefix, heads, kv, hd, page, io, in, norm, rope, hnd, fused
    ([1], [0], 16, 8, 128, 16, "f16", "f32", True, True, False, False),
    ([1] * 7, [0, 5, 15, 16, 63, 64, 1000], 32, 8, 128, 64, "bf16", "f32", True, True, False, False),
    ([3, 0, 130, 1, 0], [0, 9, 62, 255, 0], 4, 2, 64, 16, "bf16", "bf16", True, True, True, True),
    ([200], [100], 5, 1, 128, 256, "f16", "f16", False, True, False, True),
    ([33, 40], [0, 1], 3, 3, 64, 32, "f16", "f32", True, False, True, True),
    ([64, 2], [0, 77], 16, 1, 128, 128, "bf16", "f32", False, False, False, False),
    ([1, 1, 1], [3, 4, 5], 12, 4, 64, 64, "bf16", "f16", True, True, False, False),
    ([1] * 70, list(range(70)), 8, 8, 128, 16, "bf16", "f32", True, True, False, True),
    ([900, 1, 300], [0, 9, 50], 32, 8, 128, 64, "f16", "f16", True, True, False, True),  # several steps a warp
    ([700, 500], [3, 0], 7, 7, 64, 64, "bf16", "f32", True, True, True, False),
]


def codes_close(codes, scales, want, d):
    """codes * scales against rows `want` [.., dim] whose exact scales are d."""
    assert float(((scales.double() - d).abs() / d).max()) <= 2.0 ** -20
    x = want / d[..., None]
    tol = torch.clamp(x.abs() * 2.0 ** -4, min=2.0 ** -10) + 448 * 2.0 ** -19 * 1.1
    over = (codes.double() - x).abs() - tol
    assert float(over.max()) <= 0, float(over.max())


@pytest.mark.parametrize("new,pre,H,kv,hd,page,io,inp,norm,rope,hnd,fused", APPEND)
def test_append(new, pre, H, kv, hd, page, io, inp, norm, rope, hnd, fused):
    g = gen(len(new) * hd + page)
    lens = [a + b for a, b in zip(new, pre)]
    n = sum(new)
    rows, pages = ids_of(g, [-(-m // page) for m in lens])
    k, v, scales = pool8(g, pages, page, kv, hd, hnd)
    it = {"f32": torch.float32, **DT}[inp]
    if fused:
        x = randn(g, n, H + 2 * kv, hd, dtype=it)
        q, kn, vn = x[:, :H], x[:, H:H + kv], x[:, H + kv:]
    else:
        q, kn, vn = randn(g, n, H, hd, dtype=it), randn(g, n, kv, hd, dtype=it), randn(g, n, kv, hd, dtype=it)
    qg, kg = (1 + 0.1 * randn(g, hd), 1 + 0.1 * randn(g, hd)) if norm else (None, None)
    tab = rb.rope_table(max(lens) + 1, hd) if rope else None
    cu = [0] + np.cumsum(new).tolist()
    cache = rb.PagedKV8(k, v, scales, dtype=DT[io])
    batch = rb.PagedBatch(i32(padded(rows)), i32(lens), i32(cu), n)
    k0, v0, s0 = k.view(torch.uint8).clone(), v.view(torch.uint8).clone(), scales.clone()
    got = rb.paged_append(cache, batch, q, kn, vn, qg, kg, 1e-6, tab)
    pos = torch.tensor([lens[s] - m + i for s, m in enumerate(new) for i in range(m)], device="cuda")
    at = [(rows[s][(lens[s] - m + i) // page], (lens[s] - m + i) % page) for s, m in enumerate(new) for i in range(m)]
    pg, sl = (torch.tensor([a[i] for a in at], device="cuda") for i in (0, 1))
    wq = turned(q, qg, tab, pos, 1e-6)
    u = U[DT[io]]
    big = wq.abs().amax(-1, keepdim=True)
    assert got.dtype is DT[io] and bool(((got.double() - wq).abs() <= u * wq.abs() * 1.01 + 2.0 ** -19 * big).all())
    for pool, raw, x, gain, r, which in ((k, k0, kn, kg, tab, 0), (v, v0, vn, None, None, 1)):
        want = turned(x, gain, r, pos, 1e-6)
        d = (want.abs().amax(-1) / 448).clamp(min=2.0 ** -126)
        codes_close(pool.view(torch.uint8)[pg, sl].view(E4M3), scales[pg, :, which, sl], want, d)
        now = pool.view(torch.uint8).clone()
        now[pg, sl] = raw[pg, sl]
        assert torch.equal(now, raw)  # nothing else is written
    now = scales.clone()
    now[pg, :, :, sl] = s0[pg, :, :, sl]
    assert torch.equal(now, s0)


@pytest.mark.parametrize("hd", [64, 128])
def test_append_rows_out_of_the_ordinary(hd):
    # zeros, tiny, huge, infinite and NaN rows; a row beside each is as it would be alone
    kv, page = 3, 16
    x = torch.ones(9, kv, hd, device="cuda") * torch.linspace(-1, 1, hd, device="cuda")
    x[0, 1] = 0
    x[1, 1] *= 1e-41  # subnormal
    x[2, 1] *= 3e38
    x[3, 1, 5] = float("inf")
    x[4, 1, hd - 1] = float("-inf")
    x[5, 1, 0] = float("nan")
    x[6, 1] *= 2.0 ** -120
    x[7, 1] = 0
    x[7, 1, hd // 2] = -2.5
    cache = rb.PagedKV8.empty(2, page, kv, hd, torch.float16)
    batch = rb.PagedBatch(i32([[1]]), i32([9]), i32([0, 9]), 9)
    assert rb.paged_append(cache, batch, None, x, -x) is None
    k, v, sc = cache.k[1, :9].float(), cache.v[1, :9].float(), cache.scales[1, :, :, :9].permute(2, 0, 1)
    assert float(k[0, 1].abs().max()) == 0 and bool((sc[0, 1] == 2.0 ** -126).all())
    assert bool((sc[1, 1] == 2.0 ** -126).all())
    for i in (3, 4, 5):
        assert bool(sc[i, 1].isnan().all()) and bool((k[i, 1] * sc[i, 1, 0]).isnan().all())
    want = x.double()
    for i in (1, 2, 6, 7, 8):
        d = (want[i, 1].abs().max() / 448).clamp(min=2.0 ** -126)
        codes_close(k[i, 1], sc[i, 1, 0], want[i, 1], d)
        codes_close(v[i, 1], sc[i, 1, 1], -want[i, 1], d)
    assert bool((k[:, 0] == k[8, 0]).all()) and bool((sc[:, 0] == sc[8, 0]).all()) and bool((k[:, 2] == k[8, 2]).all())


def test_append_drops_what_has_no_place():
    kv, hd, page = 2, 64, 16
    cache = rb.PagedKV8.empty(3, page, kv, hd)
    for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.scales):
        t.fill_(7)
    before = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.scales)]
    g = gen(1)
    status = i32([0])
    q, k, v = randn(g, 6, 4, hd), randn(g, 6, kv, hd), randn(g, 6, kv, hd)
    # page ids outside the pool, a position past the table, rows of no sequence
    batch = rb.PagedBatch(i32([[3], [-1], [1]]), i32([1, 1, 17]), i32([1, 2, 3, 4]), 6, status)
    got = rb.paged_append(cache, batch, q, k, v)
    assert float(got.float().abs().max()) == 0 and int(status) == paged.DROPPED
    for t, b in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.scales), before):
        assert torch.equal(t, b)


# -------------------------------------------------------------- reading back
READ = [  # lengths, kv, hd, page, to page, io, hnd, to hnd
    ([1], 1, 64, 16, 16, "f16", False, False),
    ([33, 0, 16, 1, 500], 8, 128, 16, 64, "bf16", False, True),
    ([255, 256, 257], 3, 64, 256, 16, "f16", True, False),
    ([3000, 7, 0, 0], 8, 128, 64, 128, "bf16", True, True),
    ([i % 40 for i in range(90)], 2, 128, 32, 32, "f16", False, False),
]


@pytest.mark.parametrize("lens,kv,hd,page,to_page,io,hnd,to_hnd", READ)
def test_read(lens, kv, hd, page, to_page, io, hnd, to_hnd):
    g = gen(sum(lens) + hd)
    rows, pages = ids_of(g, [-(-n // page) for n in lens])
    to_rows, to_pages = ids_of(g, [-(-n // to_page) for n in lens])
    k, v, scales = pool8(g, pages, page, kv, hd, hnd)
    to = pool16(g, to_pages, to_page, kv, hd, DT[io], to_hnd)
    want = [t.clone() for t in to]
    cache = rb.PagedKV8(k, v, scales, dtype=DT[io])
    for s, n in enumerate(lens):
        for t in range(n):
            src, dst = (rows[s][t // page], t % page), (to_rows[s][t // to_page], t % to_page)
            for w, pool, x in ((0, k, want[0]), (1, v, want[1])):
                x[dst] = (pool[src].float() * scales[src[0], :, w, src[1], None]).to(DT[io])
    assert rb.paged_read(cache, rb.PagedBatch(i32(padded(rows)), i32(lens)), rb.PagedKV(*to), i32(padded(to_rows))) is None
    assert torch.equal(to[0], want[0]) and torch.equal(to[1], want[1])


def test_read_leaves_out_what_is_not_there():
    # source pages that are not there keep their slots; places that are not there drop
    kv, hd, page = 2, 64, 16
    g = gen(3)
    k, v, scales = pool8(g, 5, page, kv, hd)
    scales[4] = float("nan")  # a row that was not finite
    to = pool16(g, 6, page, kv, hd, torch.float16)
    want = [t.clone() for t in to]
    cache = rb.PagedKV8(k, v, scales, dtype=torch.float16)
    status = i32([0])
    batch = rb.PagedBatch(i32([[0, -1, 5, 1], [2, 3, -1, -1], [4, -1, -1, -1]]), i32([60, 100, -3]), status=status)
    rb.paged_read(cache, batch, rb.PagedKV(*to), i32([[0, 1, 2, 3], [4, 5, -1, -1], [0, 0, 0, 0]]))
    for w, pool, x in ((0, k, want[0]), (1, v, want[1])):
        val = (pool.float() * scales[:, :, w].transpose(1, 2)[..., None]).half()
        x[0], x[3, :12], x[4], x[5] = val[0], val[1, :12], val[2], val[3]
    assert torch.equal(to[0], want[0]) and torch.equal(to[1], want[1]) and int(status) == 0
    # no page in to_table; a table shorter than the sequence; ids outside the pool
    for tab, kept in (([[5, -1]], 16), ([[5]], 16), ([[5, 6]], 16), ([[5, 4]], 20)):
        status.zero_()
        rb.paged_read(cache, rb.PagedBatch(i32([[2, 3]]), i32([20]), status=status), rb.PagedKV(*to), i32(tab))
        assert int(status) == (0 if kept == 20 else paged.DROPPED)
    one = rb.PagedBatch(i32([[4]]), i32([1]))
    rb.paged_read(cache, one, rb.PagedKV(*to), i32([[0]]))
    assert bool(to[0][0, 0].isnan().all()) and not bool(to[0][0, 1].isnan().any())


# -------------------------------------------------- single-token attention
def own_cache(g, kind, pages, page, kv, hd, io, hnd):
    if kind == "e4m3":
        return rb.PagedKV8(*pool8(g, pages, page, kv, hd, hnd), dtype=DT[io])
    return rb.PagedKV(*pool16(g, pages, page, kv, hd, DT[io], hnd))


DECODE = [  # lengths, heads, kv, hd, page, io, hnd
    ([1], 16, 8, 128, 16, "f16", False),
    ([33], 16, 8, 128, 16, "f16", False),
    ([0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200], 32, 8, 128, 64, "bf16", False),
    ([4200], 32, 8, 128, 64, "bf16", False),
    ([777, 5, 0, 3000], 8, 8, 128, 128, "f16", True),
    ([100, 1000, 31], 12, 4, 64, 32, "bf16", True),
    ([1, 2, 500, 64], 12, 12, 64, 16, "f16", False),
    ([300, 41], 5, 1, 128, 256, "bf16", False),
    ([2000, 0, 13], 16, 1, 64, 64, "f16", True),
    ([900, 61], 32, 2, 128, 64, "bf16", False),  # groups of 16
    ([i % 50 for i in range(200)], 9, 1, 64, 16, "bf16", False),
    ([129] * 40, 32, 8, 128, 16, "f16", False),
]


@pytest.mark.parametrize("lens,H,kv,hd,page,io,hnd", DECODE)
def test_decode_over_8_bits(lens, H, kv, hd, page, io, hnd):
    g = gen(sum(lens) + H)
    rows, pages = ids_of(g, [-(-n // page) for n in lens])
    cache = own_cache(g, "e4m3", pages, page, kv, hd, io, hnd)
    q = randn(g, len(lens), H, hd, dtype=DT[io])
    batch = rb.PagedBatch(i32(padded(rows)), i32(lens))
    got = rb.paged_attention_decode(cache, batch, q)
    close(got, *definition(cache, rows, lens, q, hd ** -0.5))
    for _ in range(3):  # the same bits again
        assert torch.equal(rb.paged_attention_decode(cache, batch, q), got)


SHARED = [  # own lengths (None: no positions at all), prefixes, cu, heads, kv, hd, page, io, hnd
    ([1, 2, 3, 4], [40], [0, 4], 8, 2, 128, 16, "bf16", False),
    ([10] * 9, [300], [0, 9], 32, 8, 128, 64, "bf16", False),
    ([0, 0, 7], [64], [0, 3], 16, 8, 128, 64, "f16", False),  # nothing but the prefix
    ([5, None, 70, 130, None], [1, 17], [0, 2, 5], 12, 4, 64, 16, "f16", True),
    ([64, 65, 1], [0, 1000], [0, 1, 3], 16, 1, 128, 128, "bf16", True),  # an empty prefix
    ([3] * 5, [200, 100, 50], [0, 2, 2, 3], 5, 1, 64, 32, "f16", False),  # an empty group, sequences in none
    ([20] * 6, [130], [2, 5], 8, 8, 64, 64, "bf16", False),  # sequences before and behind the group
    ([i % 9 for i in range(70)], [129], [0, 70], 8, 2, 128, 16, "f16", False),
    ([i % 30 for i in range(200)], [2000, 500, 31], [0, 100, 150, 190], 16, 8, 128, 64, "bf16", False),
    ([400, 1], [4096], [0, 2], 32, 8, 128, 256, "bf16", True),
    ([2, 300], [700], [0, 2], 32, 2, 128, 64, "f16", False),  # groups of 16
    ([17] * 33, [515], [0, 33], 9, 1, 64, 32, "bf16", False),
    ([1] * 300, [256], [0, 300], 4, 1, 128, 64, "bf16", False),
]


NONE = 16  # groups without a sequence, after those of "many"
KINDS = pytest.mark.parametrize("kind", ["same", "other", "many", "e4m3"])


def shared_case(own, plens, cu, H, kv, hd, page, io, hnd, kind, seed=0):
    """kind: "same" (16 bits, the prefix in the sequences' own pool), "other" (16 bits, the prefix
    in a pool of other pages), "many" (as "same", among so many groups that a plan is made) or "e4m3"."""
    if kind == "many" and plens:
        plens, cu = plens + [0] * NONE, cu + [cu[-1]] * NONE
    ppage = (16 if page > 16 else 64) if kind == "other" else page
    g = gen(len(own) * hd + sum(plens) + seed)
    group = [next((j for j in range(len(plens)) if cu[j] <= s < cu[j + 1]), -1) for s in range(len(own))]
    lens = [0 if n is None else n + (plens[j] if j >= 0 else 0) for n, j in zip(own, group)]
    held = [plens[j] // page if j >= 0 else 0 for j in group]
    need = [max(0, -(-n // page) - h) for n, h in zip(lens, held)]
    rows, pages = ids_of(g, [-(-p // ppage) for p in plens] + need)
    first, mine = rows[:len(plens)], rows[len(plens):]
    cache = own_cache(g, "e4m3" if kind == "e4m3" else "16", pages, page, kv, hd, io, hnd)
    pre = cache if kind in ("same", "many") else own_cache(g, "16", pages, ppage, kv, hd, io, hnd != (kind == "other"))
    # (their own tables do not have the prefix's positions at all)
    table = [[-1] * h + r for h, r in zip(held, mine)]
    q = randn(g, len(own), H, hd, dtype=DT[io])
    batch = rb.PagedBatch(i32(padded(table)), i32(lens))
    prefix = rb.PagedPrefix(pre, i32(padded(first)), i32(plens), i32(cu)) if plens else None
    return cache, batch, prefix, q, table, lens, (pre, first, plens, cu)


@KINDS
@pytest.mark.parametrize("own,plens,cu,H,kv,hd,page,io,hnd", SHARED)
def test_decode_with_a_shared_prefix(own, plens, cu, H, kv, hd, page, io, hnd, kind):
    cache, batch, prefix, q, table, lens, pre = shared_case(own, plens, cu, H, kv, hd, page, io, hnd, kind)
    got = rb.paged_attention_decode(cache, batch, q, prefix=prefix)
    close(got, *definition(cache, table, lens, q, hd ** -0.5, pre))
    for _ in range(3):
        assert torch.equal(rb.paged_attention_decode(cache, batch, q, prefix=prefix), got)


@pytest.mark.parametrize("kind", ["same", "many", "e4m3"])
def test_sequences_shorter_than_their_prefix(kind):
    # they see as much of it as they have positions; pages that are not there, in the
    # prefix and behind it; a prefix longer than its table, a length below zero
    own, plens, cu = [30] * 8, [200, 100], [0, 6, 8]
    cache, batch, prefix, q, table, lens, pre = shared_case(own, plens, cu, 8, 2, 128, 16, "bf16", False, kind)
    lens = [230, 1, 199, 200, 201, 16, -5, 130]
    first = [r[:] for r in pre[1]]
    first[0][3], first[0][7] = -1, 10 ** 6
    table = [r[:] for r in table]
    table[0][13] = -1
    table[7] = table[7][:7]
    plens = [200, 1000]
    first[1] = first[1][:5]  # positions 80 .. are past what its row names
    width = max(len(r) for r in first)
    first[1] += [-1] * (width - 5)
    batch = rb.PagedBatch(i32(padded(table)), i32(lens))
    plens, cu = plens + pre[2][2:], pre[3]
    prefix = rb.PagedPrefix(pre[0], i32(padded(first)), i32(plens), i32(cu))
    got = rb.paged_attention_decode(cache, batch, q, prefix=prefix)
    close(got, *definition(cache, table, lens, q, 128 ** -0.5, (pre[0], first, plens, cu)))


def test_a_prefix_without_groups_is_none():
    own = [30, 1, 0, 200]
    cache, batch, _, q, table, lens, pre = shared_case(own, [], [0], 8, 2, 64, 16, "f16", False, "same")
    empty = rb.PagedPrefix(pre[0], torch.zeros(0, 3, dtype=torch.int32, device="cuda"), i32([]), i32([0]))
    got = rb.paged_attention_decode(cache, batch, q, prefix=empty)
    close(got, *definition(cache, table, lens, q, 64 ** -0.5))


@KINDS
@pytest.mark.parametrize("hd", [64, 128])
def test_what_nobody_sees_is_never_used(kind, hd):
    # every slot that no sequence sees: NaN, infinities, codes and scales that are NaN
    own, plens, cu = [1, 37, 64, 0, 90], [70, 33], [0, 3, 4]
    cache, batch, prefix, q, table, lens, pre = shared_case(own, plens, cu, 8, 2, hd, 32, "bf16", False, kind)
    want = rb.paged_attention_decode(cache, batch, q, prefix=prefix)
    used = torch.zeros(cache.k.shape[:2], dtype=torch.bool, device="cuda")
    pused = used if kind in ("same", "many") else torch.zeros(pre[0].k.shape[:2], dtype=torch.bool, device="cuda")
    size = pused.shape[1]
    group = [0, 0, 0, 1, -1]
    for s, n in enumerate(lens):
        for t in range(plens[group[s]] if group[s] >= 0 else 0, n):
            used[table[s][t // 32], t % 32] = True
    for j, p in enumerate(plens):
        for t in range(p):
            pused[pre[1][j][t // size], t % size] = True
    for bad in (float("nan"), float("inf"), -3e38):
        pre[0].k[~pused], pre[0].v[~pused] = bad, bad
        if kind == "e4m3":
            for t in (cache.k, cache.v):
                t.view(torch.uint8)[~used] = 0x7F if bad != bad else 0x7E
            cache.scales.permute(0, 3, 1, 2)[~used] = bad
        elif kind == "other":
            cache.k[~used], cache.v[~used] = bad, bad
        assert torch.equal(rb.paged_attention_decode(cache, batch, q, prefix=prefix), want)


@KINDS
def test_values_that_are_not_finite_show(kind):
    own, plens, cu = [40, 40, 40, 40], [100], [0, 2]
    cache, batch, prefix, q, table, lens, pre = shared_case(own, plens, cu, 4, 2, 64, 16, "bf16", False, kind)
    want = rb.paged_attention_decode(cache, batch, q, prefix=prefix)
    # an own position of sequence 0, kv head 1
    t = 105
    at = table[0][t // 16], t % 16
    if kind != "e4m3":
        cache.v[at[0], at[1], 1, 3] = float("inf")
    else:
        cache.scales[at[0], 1, 1, at[1]] = float("nan")
    got = rb.paged_attention_decode(cache, batch, q, prefix=prefix)
    if kind != "e4m3":
        assert bool((got[0, 2:, 3] == float("inf")).all())
        assert torch.isfinite(got[0, 2:, :3]).all() and torch.isfinite(got[0, 2:, 4:]).all()
    else:
        assert bool(got[0, 2:].isnan().all())
    assert torch.equal(got[0, :2], want[0, :2]) and torch.equal(got[1:], want[1:])
    # a position of the prefix, kv head 0: all of its group
    pre[0].v[pre[1][0][1 if kind == "other" else 2], 7, 0, 5] = float("-inf")
    got2 = rb.paged_attention_decode(cache, batch, q, prefix=prefix)
    assert bool((got2[:2, :2, 5] == float("-inf")).all()) and torch.isfinite(got2[:2, :2, :5]).all()
    assert torch.equal(got2[2:], want[2:]) and torch.equal(got2[1, 2:], want[1, 2:])
    # a query that is NaN
    q[3, 1] = float("nan")
    got3 = rb.paged_attention_decode(cache, batch, q, prefix=prefix)
    assert bool(got3[3, 1].isnan().all()) and torch.equal(got3[3, 0], got2[3, 0]) and torch.equal(got3[2], got2[2])


@KINDS
@pytest.mark.parametrize("io", ["bf16", "f16"])
def test_scores_and_values_over_a_wide_range(kind, io):
    # scores that grow along the sequence, scales over many powers of two, large q
    own, plens, cu = [500, 3, 200], [300], [0, 2]
    cache, batch, prefix, q, table, lens, pre = shared_case(own, plens, cu, 8, 2, 128, 64, io, False, kind)
    ramp = torch.exp2(torch.arange(cache.k.shape[0], device="cuda").float() % 7 - 3)
    if kind == "e4m3":
        cache.scales.mul_(ramp[:, None, None, None])
    else:
        for t in (cache.k, cache.v):
            t.copy_((t.float() * ramp[:, None, None, None]).to(t.dtype))
    for mul in (1.0, 30.0, 2.0 ** -12):
        q2 = (q.float() * mul).to(q.dtype)
        got = rb.paged_attention_decode(cache, batch, q2, prefix=prefix)
        close(got, *definition(cache, table, lens, q2, 128 ** -0.5, pre))


# ------------------------------------------------------ calls as they are made
def test_strides_scale_and_out():
    g = gen(9)
    lens, H, kv, hd, page = [70, 3], 8, 2, 128, 16
    rows, pages = ids_of(g, [5, 1])
    k, v, scales = pool8(g, pages, page, 2 * kv, hd)
    wide = torch.zeros(pages, 2 * kv, 3, page, device="cuda")[:, :, :2]
    wide.copy_(scales)
    cache = rb.PagedKV8(k[:, :, 1::2], v[:, :, 1::2], wide[:, 1::2], dtype=torch.float16)  # every other head of a wider pool
    q = randn(g, 2, 2 * H, hd, dtype=torch.float16)[:, ::2]
    out = torch.empty(2, H, hd, dtype=torch.float16, device="cuda")
    got = rb.paged_attention_decode(cache, rb.PagedBatch(i32(padded(rows)), i32(lens)), q, scale=0.3, out=out)
    assert got is out
    close(got, *definition(cache, rows, lens, q, 0.3))


@KINDS
def test_captured_calls_follow_lengths_and_tables(kind):
    own, plens, cu = [30, 5, 0, 99], [150], [0, 3]
    cache, batch, prefix, q, table, lens, pre = shared_case(own, plens, cu, 8, 2, 128, 16, "bf16", False, kind)
    rb.paged_attention_decode(cache, batch, q, prefix=prefix)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rb.paged_attention_decode(cache, batch, q, prefix=prefix)
    for plen, n, c in ((150, [180, 155, 150, 99], [0, 3]), (64, [170, 64, 1, 50], [1, 2]), (0, [4, 5, 6, 7], [0, 4]), (150, [0, 0, 0, 0], [0, 4])):
        plens, c = [plen] + pre[2][1:], c + c[-1:] * (len(pre[3]) - 2)
        batch.keep[1].copy_(i32(n))
        prefix.keep[1].copy_(i32(plens))
        prefix.keep[2].copy_(i32(c))
        graph.replay()
        tab = [[x if x >= 0 else -1 for x in r] for r in table]
        close(got, *definition(cache, tab, n, q, 128 ** -0.5, (pre[0], pre[1], plens, c)))


@pytest.mark.parametrize("kind", ["same", "many"])
def test_two_streams_at_once(kind):
    own, plens, cu = [300 + i for i in range(6)], [2000], [0, 6]
    cache, batch, prefix, q, *_ = shared_case(own, plens, cu, 32, 8, 128, 64, "bf16", False, kind)
    want = rb.paged_attention_decode(cache, batch, q, prefix=prefix)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got += [rb.paged_attention_decode(cache, batch, q, prefix=prefix) for _ in range(4)]
            got.append(rb.paged_attention_decode(cache, batch, q, prefix=prefix, stream=s.cuda_stream))
        torch.cuda.synchronize()
        assert all(torch.equal(x, want) for x in got)


def test_a_step_of_many_conversations():
    # an opening enters in 8 bits, is read back once, prompts continue it, then steps
    # decode over both; against the same calls on one 16-bit cache of the values held
    H, kv, hd, page, open_, own = 8, 2, 128, 16, 90, [5, 17, 33]
    g, S = gen(4), len(own)
    rb.paged_status()  # (what earlier calls have reported)
    rope = rb.rope_table(256, hd)
    per = 10
    c8 = rb.PagedKV8.empty(S * per + 6, page, kv, hd, torch.bfloat16)
    x = [randn(g, open_, h, hd) for h in (H, kv, kv)]
    rb.paged_append(c8, rb.PagedBatch(i32([list(range(6))]), i32([open_]), i32([0, open_]), open_), *x, rope=rope)
    pre = rb.PagedKV.empty(6, page, kv, hd, torch.bfloat16)
    rb.paged_read(c8, rb.PagedBatch(i32([list(range(6))]), i32([open_])), pre, i32([[5, 4, 3, 2, 1, 0]]))
    rows = [[6 + s * per + j for j in range(per)] for s in range(S)]
    lens, n = [open_ + m for m in own], sum(own)
    cu = [0] + np.cumsum(own).tolist()
    x = [randn(g, n, h, hd) for h in (H, kv, kv)]
    table = i32(rows)
    q = rb.paged_append(c8, rb.PagedBatch(table, i32(lens), i32(cu), n), *x, rope=rope)
    # the prompts: a 16-bit scratch pool with the opening and what was just written
    scratch = rb.PagedKV.empty(S * per + 6, page, kv, hd, torch.bfloat16)
    whole = i32([[0, 1, 2, 3, 4] + r[5:] for r in rows])  # (the opening's last, unfilled page is the conversations' own)
    opening = rb.PagedBatch(i32([list(range(6))] * S), i32([open_] * S))
    rb.paged_read(c8, rb.PagedBatch(table, i32(lens)), scratch, table)
    rb.paged_read(c8, opening, scratch, i32([[0, 1, 2, 3, 4, r[5]] for r in rows]))
    got = rb.paged_attention_prompt(scratch, rb.PagedBatch(whole, i32(lens), i32(cu), n), q)
    assert torch.isfinite(got).all()
    step = rb.PagedBatch(table, i32(lens))
    prefix = rb.PagedPrefix(pre, i32([[5, 4, 3, 2, 1, 0]]), i32([open_]), i32([0, S]))
    for _ in range(3):
        step.keep[1].add_(1)
        lens = [m + 1 for m in lens]
        x = [randn(g, S, h, hd) for h in (H, kv, kv)]
        q = rb.paged_append(c8, step, *x, rope=rope)
        got = rb.paged_attention_decode(c8, step, q, prefix=prefix)
        close(got, *definition(c8, rows, lens, q, hd ** -0.5, (pre, [[5, 4, 3, 2, 1, 0]], [open_], [0, S])))
    assert rb.paged_status() == 0
