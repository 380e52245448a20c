"""Shared prefixes at sizes where the work is cut in many ways, against the same call
without a prefix.

Both are within 1.25 u (|e| + sum p |v|) of the exact value e (test_gpu_paged8.py has the
terms; u = 2^-8 for bfloat16, 2^-11 for float16), and so within 2.5 u (|e| + sum p |v|) of
each other; sum p |v| is what the call without a prefix gives over |v|, itself within
1.25 u (1 + 1) of it, so 1.02 times that covers it.
"""
import random

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import rpgbarengine_b200 as rb  # noqa: E402

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
    if not torch.cuda.is_available() or rb.device_count() == 0:
        pytest.fail("GPU test collected without a CUDA device")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def case(n_seqs, groups, plen, own, H, kv, hd, page, io, seed=0, loose=0, empty=0):
    """Sequences whose tables name their group's pages, then their own: with and without a
    prefix the calls see the same.  plen, own: (from, to), prefixes in whole pages."""
    r = random.Random(seed)
    n = n_seqs - loose
    cu = [0] + sorted(r.sample(range(1, n), groups - 1)) + [n]
    plens = [r.randint(plen[0] // page, plen[1] // page) * page for _ in range(groups)]
    at, first = 0, []
    for p in plens:
        first.append(list(range(at, at + p // page)))
        at += p // page
    rows, lens, g = [], [], 0
    for s in range(n_seqs):
        while g < groups and s >= cu[g + 1]:
            g += 1
        mine = first[g] if s < n else []
        k = 0 if empty and s % empty == empty - 1 else r.randint(*own)
        more = -(-k // page)
        rows.append(mine + list(range(at, at + more)))
        at += more
        lens.append(0 if empty and s % empty == empty - 1 else len(mine) * page + k)
    width = max(1, max(len(x) for x in rows))
    table = i32([x + [-1] * (width - len(x)) for x in rows])
    pw = max(1, max(len(x) for x in first))
    ptable = i32([x + [-1] * (pw - len(x)) for x in first])
    gen = torch.Generator(device="cuda").manual_seed(seed)
    k, v = (torch.randn(at + 1, page, kv, hd, generator=gen, device="cuda", dtype=DT[io]) for _ in range(2))
    q = torch.randn(n_seqs, H, hd, generator=gen, device="cuda", dtype=DT[io])
    return k, v, q, table, i32(lens), ptable, i32(plens), i32(cu)


def check(k, v, q, table, lens, ptable, plens, cu):
    cache, batch = rb.PagedKV(k, v), rb.PagedBatch(table, lens)
    prefix = rb.PagedPrefix(cache, ptable, plens, cu)
    got = rb.paged_attention_decode(cache, batch, q, prefix=prefix)
    want = rb.paged_attention_decode(cache, batch, q)
    mag = rb.paged_attention_decode(rb.PagedKV(k, v.abs()), batch, q).double()
    assert torch.isfinite(got).all()
    over = (got.double() - want.double()).abs() - 2.5 * U[q.dtype] * (want.double().abs() + 1.02 * mag)
    assert float(over.max()) <= 0, float(over.max())
    for _ in range(2):
        assert torch.equal(rb.paged_attention_decode(cache, batch, q, prefix=prefix), got)
    return cache, batch, prefix, got


CASES = [
    dict(n_seqs=2, groups=1, plen=(9008, 9008), own=(1, 40), H=1, kv=1, hd=64, page=16, io="bf16"),  # as many pieces as there are
    dict(n_seqs=3, groups=1, plen=(256, 256), own=(20000, 20000), H=8, kv=2, hd=128, page=64, io="f16"),  # items that many CTAs share
    dict(n_seqs=1, groups=1, plen=(128, 128), own=(130000, 130000), H=4, kv=1, hd=64, page=128, io="bf16"),
    dict(n_seqs=90, groups=40, plen=(0, 700), own=(0, 90), H=16, kv=8, hd=128, page=16, io="bf16"),  # more units than CTAs
    dict(n_seqs=700, groups=33, plen=(64, 2000), own=(1, 30), H=4, kv=1, hd=64, page=32, io="f16", loose=5),
    dict(n_seqs=3000, groups=1500, plen=(0, 64), own=(0, 20), H=2, kv=1, hd=64, page=16, io="bf16", empty=7),  # look-ups outside shared memory
    dict(n_seqs=5000, groups=2, plen=(16, 300), own=(0, 33), H=2, kv=2, hd=64, page=16, io="f16", loose=100),
    dict(n_seqs=1025, groups=1024, plen=(16, 48), own=(1, 5), H=4, kv=4, hd=128, page=16, io="bf16"),
    dict(n_seqs=300, groups=1, plen=(8192, 8192), own=(1, 3), H=32, kv=8, hd=128, page=256, io="bf16"),
    dict(n_seqs=64, groups=64, plen=(16, 1000), own=(1, 1), H=12, kv=12, hd=64, page=16, io="f16"),  # groups of one
    dict(n_seqs=130, groups=3, plen=(100, 3000), own=(0, 600), H=16, kv=1, hd=128, page=64, io="f16", empty=3),
]


@pytest.mark.parametrize("c", CASES, ids=lambda c: f"{c['n_seqs']}x{c['groups']}")
def test_with_and_without_a_prefix(c):
    check(*case(**c, seed=c["n_seqs"] + c["groups"]))


FEW = [
    dict(n_seqs=1, groups=1, plen=(16, 16), own=(0, 0), H=1, kv=1, hd=64, page=16, io="f16"),  # half a warp of output
    dict(n_seqs=7, groups=2, plen=(16, 700), own=(0, 1), H=3, kv=3, hd=64, page=16, io="bf16", empty=3),
    dict(n_seqs=64, groups=1, plen=(256, 256), own=(0, 900), H=32, kv=8, hd=128, page=64, io="bf16", loose=3),
    dict(n_seqs=5, groups=4, plen=(32, 1000), own=(1, 9000), H=8, kv=2, hd=128, page=32, io="f16", loose=1),
    dict(n_seqs=512, groups=3, plen=(128, 128), own=(0, 70), H=2, kv=2, hd=64, page=128, io="bf16", empty=5),
    dict(n_seqs=40, groups=2, plen=(64, 1200), own=(0, 500), H=32, kv=2, hd=128, page=64, io="f16", empty=9),
    dict(n_seqs=60, groups=15, plen=(0, 90), own=(0, 200), H=8, kv=4, hd=64, page=16, io="f16", loose=4),
    dict(n_seqs=60, groups=16, plen=(0, 90), own=(0, 200), H=8, kv=4, hd=64, page=16, io="f16", loose=4),
    dict(n_seqs=33, groups=3, plen=(0, 400), own=(3, 300), H=16, kv=1, hd=64, page=16, io="bf16", loose=2),
]


@pytest.mark.parametrize("c", FEW, ids=lambda c: f"{c['n_seqs']}x{c['groups']}-{c['H']}-{c['kv']}-{c['hd']}")
def test_few_groups_and_the_same_beside_groups_of_none(c):
    # groups without a sequence change no result, though the call takes other kernels with them
    # (16 bits) or cuts the work another way (own positions in 8)
    k, v, q, table, lens, ptable, plens, cu = case(**c, seed=c["n_seqs"])
    none = (torch.cat([ptable, ptable.new_full((16, ptable.shape[1]), -1)]), torch.cat([plens, plens[:1].expand(16) * 0 + 32]),
            torch.cat([cu, cu[-1:].expand(16)]))
    check(k, v, q, table, lens, ptable, plens, cu)
    cache, batch, _, _ = check(k, v, q, table, lens, *none)
    ones = torch.ones(k.shape[0], c["kv"], 2, c["page"], device="cuda")
    kc, vc = k.float().to(torch.float8_e4m3fn), v.float().to(torch.float8_e4m3fn)
    c8, mags = (rb.PagedKV8(kc, x, ones, dtype=k.dtype) for x in (vc, vc.float().abs().to(torch.float8_e4m3fn)))
    few, many = (rb.PagedPrefix(cache, *x) for x in ((ptable, plens, cu), none))
    a, b = (rb.paged_attention_decode(c8, batch, q, prefix=x) for x in (few, many))
    mag = rb.paged_attention_decode(mags, batch, q, prefix=rb.PagedPrefix(rb.PagedKV(k, v.abs()), *none)).double()
    assert torch.isfinite(a).all()
    assert float(((a.double() - b.double()).abs() - 2.5 * U[q.dtype] * (b.double().abs() + 1.02 * mag)).max()) <= 0
    for _ in range(3):
        assert torch.equal(rb.paged_attention_decode(c8, batch, q, prefix=few), a)


@pytest.mark.parametrize("groups", [1, 20])
def test_a_prefix_longer_than_its_table(groups):
    # positions without a page are left out
    k, v, q, table, lens, ptable, plens, cu = case(40, groups, (64, 64), (0, 1), 4, 2, 64, 16, "bf16", seed=2)
    cache, out = rb.PagedKV(k, v), torch.full((40, 4, 64), 9.0, device="cuda", dtype=torch.bfloat16)
    for width in (1, 3):
        rb.paged_attention_decode(cache, rb.PagedBatch(table, lens), q, out=out, prefix=rb.PagedPrefix(cache, ptable[:, :width].contiguous(), plens, cu))
        t = table.clone()
        t[:, width:4] = -1
        want = rb.paged_attention_decode(cache, rb.PagedBatch(t, lens), q).double()
        mag = rb.paged_attention_decode(rb.PagedKV(k, v.abs()), rb.PagedBatch(t, lens), q).double()
        assert float(((out.double() - want).abs() - 2.5 * 2.0 ** -8 * (want.abs() + 1.02 * mag)).max()) <= 0


@pytest.mark.parametrize("io", ["bf16", "f16"])
def test_huge_values_in_a_prefix_that_is_all(io):
    # three heads of 64: the last warp has half its rows
    k, v, q, table, lens, ptable, plens, cu = case(5, 2, (64, 320), (0, 0), 3, 1, 64, 32, io, seed=4)
    for g in range(2):
        v[int(ptable[g, 0]), 5, 0, 7] = HUGE[io]
        k[int(ptable[g, 0]), 5, 0] *= 3
    got = rb.paged_attention_decode(rb.PagedKV(k, v), rb.PagedBatch(table, lens), q, prefix=rb.PagedPrefix(rb.PagedKV(k, v), ptable, plens, cu))
    assert torch.isfinite(got).all()
    for s, n in enumerate(lens.tolist()):
        K, V = (x[table[s, : n // 32].long()].reshape(-1, 64)[:n].double() for x in (k, v))
        p = torch.softmax(q[s].double() @ K.T / 8, -1)
        assert float(((got[s].double() - p @ V).abs() - 1.25 * U[DT[io]] * ((p @ V).abs() + p @ V.abs())).max()) <= 0


HUGE = {"bf16": 3.0e38, "f16": 65504.0}


@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_huge_values_in_the_prefix_and_behind_it(io, hd):
    # one value near the type's largest at a position that all see: the sums may overflow
    # on the way (weights go up to 2^40 in bfloat16), the results do not
    k, v, q, table, lens, ptable, plens, cu = case(9, 2, (64, 320), (3, 70), 8, 2, hd, 32, io, seed=3)
    for row, t in ((ptable[0], 5), (ptable[1], 63), (table[0], int(lens[0]) - 1)):
        v[int(row[t // 32]), t % 32, 1, 7] = HUGE[io]
        k[int(row[t // 32]), t % 32, 1] *= 3
    got = rb.paged_attention_decode(rb.PagedKV(k, v), rb.PagedBatch(table, lens), q, prefix=rb.PagedPrefix(rb.PagedKV(k, v), ptable, plens, cu))
    assert torch.isfinite(got).all()
    for s, n in enumerate(lens.tolist()):
        K, V = (x[table[s, : -(-n // 32)].long()].reshape(-1, 2, hd)[:n].double() for x in (k, v))
        p = torch.softmax(torch.einsum("kgd,tkd->kgt", q[s].double().view(2, -1, hd), K) * hd ** -0.5, -1)
        want, mag = (torch.einsum("kgt,tkd->kgd", p, x).reshape(8, hd) for x in (V, V.abs()))
        assert float(((got[s].double() - want).abs() - 1.25 * U[DT[io]] * (want.abs() + mag)).max()) <= 0


def test_huge_scales_in_8_bits():
    kv, hd, page = 2, 128, 16
    cache = rb.PagedKV8.empty(6, page, kv, hd, torch.bfloat16)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(50, kv, hd, generator=gen, device="cuda")
    v = torch.randn(50, kv, hd, generator=gen, device="cuda")
    v[17] *= 7e37
    v[33] *= 1e-30
    batch = rb.PagedBatch(i32([[1, 2, 3, 4]]), i32([50]), i32([0, 50]), 50)
    rb.paged_append(cache, batch, None, x, v)
    q = torch.randn(1, 8, hd, generator=gen, device="cuda", dtype=torch.bfloat16)
    got = rb.paged_attention_decode(cache, rb.PagedBatch(i32([[1, 2, 3, 4]]), i32([50])), q).double()
    K, V = ((c.view(torch.uint8)[1:5].view(torch.float8_e4m3fn).double() * cache.scales[1:5, :, w].transpose(1, 2).double()[..., None]).reshape(64, kv, hd)[:50]
            for w, c in ((0, cache.k), (1, cache.v)))
    p = torch.softmax(torch.einsum("kgd,tkd->kgt", q[0].double().view(kv, -1, hd), K) * hd ** -0.5, -1)
    want, mag = (torch.einsum("kgt,tkd->kgd", p, x).reshape(1, 8, hd) for x in (V, V.abs()))
    assert torch.isfinite(got).all() and float(((got - want).abs() - 1.25 * 2.0 ** -8 * (want.abs() + mag)).max()) <= 0


def test_calls_of_different_shapes_share_a_batch():
    # the same batch with and without a prefix, over 16 and 8 bits, in turn
    k, v, q, table, lens, ptable, plens, cu = case(20, 2, (64, 128), (1, 200), 8, 2, 128, 16, "bf16", seed=8)
    cache, batch, prefix, got = check(k, v, q, table, lens, ptable, plens, cu)
    c8 = rb.PagedKV8(k.float().to(torch.float8_e4m3fn), v.float().to(torch.float8_e4m3fn),
                     torch.ones(k.shape[0], 2, 2, 16, device="cuda"), dtype=torch.bfloat16)
    plain, eight, both = (rb.paged_attention_decode(cache, batch, q), rb.paged_attention_decode(c8, batch, q),
                          rb.paged_attention_decode(c8, batch, q, prefix=prefix))
    none = rb.PagedPrefix(cache, ptable[:0], plens[:0], cu[:1])
    for _ in range(3):
        assert torch.equal(rb.paged_attention_decode(cache, batch, q, prefix=prefix), got)
        assert torch.equal(rb.paged_attention_decode(c8, batch, q), eight)
        assert torch.equal(rb.paged_attention_decode(cache, batch, q), plain)
        assert torch.equal(rb.paged_attention_decode(c8, batch, q, prefix=prefix), both)
        assert torch.equal(rb.paged_attention_decode(cache, batch, q, prefix=none), plain)


def test_a_call_on_another_stream_sees_what_was_written_before():
    # a chain on a side stream: lengths, pages and q change right before the call, in kernels
    # that the call's first ones may overlap
    k, v, q, table, lens, ptable, plens, cu = case(40, 3, (64, 640), (20, 200), 16, 4, 128, 32, "bf16", seed=5)
    cache, batch = rb.PagedKV(k, v), rb.PagedBatch(table, lens)
    prefix = rb.PagedPrefix(cache, ptable, plens, cu)
    full = [t.clone() for t in (lens, plens, q, k)]
    want = rb.paged_attention_decode(cache, batch, q, prefix=prefix)
    side = torch.cuda.Stream()
    rb.paged_attention_decode(cache, batch, q, prefix=prefix, stream=side.cuda_stream)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for i in range(30):
            lens.copy_(full[0] - 1 - i % 3)
            plens.copy_(full[1] - 16)
            q.zero_()
            k.mul_(0.5)
            rb.paged_attention_decode(cache, batch, q, prefix=prefix)
            k.copy_(full[3])
            q.copy_(full[2])
            plens.copy_(full[1])
            lens.copy_(full[0])
            got = rb.paged_attention_decode(cache, batch, q, prefix=prefix)
            side.synchronize() if i % 10 == 9 else None
            assert torch.equal(got, want) if i % 10 == 9 else True


def test_bad_groups_stay_inside():
    # cu_seqs that decreases or leaves the batch, page ids of nowhere, lengths of any value:
    # the results may be anything, what lies beside them is not touched, and good calls after it are right
    k, v, q, table, lens, ptable, plens, cu = case(30, 3, (64, 320), (1, 90), 8, 2, 128, 16, "bf16", seed=6)
    cache, batch, prefix, want = check(k, v, q, table, lens, ptable, plens, cu)
    good = [t.clone() for t in (k, v, table, lens, ptable, plens, cu)]
    out = torch.zeros(32, 8, 128, dtype=torch.bfloat16, device="cuda")
    for bad_cu, bad_len, bad_plen in (([20, 10, 40, -5], 200, 100), ([0, 30, 0, 30], -1, 10 ** 9), ([-7, 5, 1000, 2000], 2 ** 31 - 1, -3), ([30, 30, 30, 30], 0, 64)):
        cu.copy_(i32(bad_cu))
        lens.copy_(torch.where(torch.arange(30, device="cuda") % 3 == 0, bad_len, good[3]).to(torch.int32))
        plens.copy_(i32([bad_plen, 64, 2 ** 31 - 1]))
        ptable.copy_(torch.where(torch.arange(ptable.shape[1], device="cuda") % 2 == 0, 2 ** 31 - 1, good[4]).to(torch.int32))
        if bad_len == 2 ** 31 - 1:
            lens.clamp_(max=100000)
        rb.paged_attention_decode(cache, batch, q, out=out[1:31], prefix=prefix)
        torch.cuda.synchronize()
        assert float(out[0].float().abs().max()) == 0 and float(out[31].float().abs().max()) == 0
    for t, g in zip((k, v, table, lens, ptable, plens, cu), good):
        if t is k or t is v or t is table:
            assert torch.equal(t, g)
        t.copy_(g)
    assert torch.equal(rb.paged_attention_decode(cache, batch, q, prefix=prefix), want)
