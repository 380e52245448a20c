"""Paged-cache operators at the edges of their contract.

Where two calls do the same arithmetic on the same visible values their results
are compared bit for bit; else against 64 bits with the bounds of
test_gpu_paged.py."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import rpgbarengine_b200 as rb  # noqa: E402
from test_gpu_paged import (DT, U, append_inputs, check_decode, check_packed, check_paged, decode_case, gen, i32, make_pool,  # noqa: E402
                            packed_inputs, randn)


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
    if not torch.cuda.is_available() or rb.device_count() == 0:
        pytest.fail("GPU test collected without a CUDA device")


# -------------------------------------------------------------- workspace
WORKSPACE = [  # lens, heads, kv, hd, page, cache
    ([4200], 32, 8, 128, 64, "bf16"),
    ([900 + 31 * i for i in range(64)], 32, 8, 128, 64, "bf16"),
    ([3000, 17], 12, 12, 64, 16, "f16"),
    ([2500, 1, 0, 1800], 16, 1, 128, 128, "f16"),
    ([70 + i for i in range(300)], 8, 8, 64, 32, "bf16"),
]


def test_one_workspace_serves_calls_of_every_shape():
    # a host's workspace, as large as its largest call needs and zeroed once: calls
    # of few and of many sequences, of other head counts and head sizes, in turn
    L = rb.lib()
    calls = []
    for lens, H, kv, hd, page, ty in WORKSPACE:
        k, v, table, q = decode_case(lens, H, kv, hd, page, ty, False)
        cache, batch = rb.PagedKV(k, v), rb.PagedBatch(i32(table), i32(lens))
        want = rb.paged_attention_decode(cache, batch, q)  # (a workspace of the batch's own)
        check_decode(want, q, k, v, table, lens, hd ** -0.5)
        size = L.rpgc_paged_decode_workspace(cache.ref, len(lens), H)
        assert size > 0
        calls.append((cache, batch, q, want, size))
    size = max(c[4] for c in calls)
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    for order in ((0, 1, 2, 3, 4), (4, 0, 1, 0, 4), (1, 3, 1, 2, 1, 0)):
        for i in order:
            cache, batch, q, want, _ = calls[i]
            out = torch.full_like(q, 7)
            st = rb.paged._S2(q.stride(0), q.stride(1))
            rc = L.rpgc_paged_attention_decode(cache.ref, batch.ref, q.data_ptr(), st, q.shape[1], cache.scale, out.data_ptr(),
                                               ws.data_ptr(), size, stream)
            assert rc == rb.OK
            assert torch.equal(out, want), i


# ------------------------------------------------------------ block tables
def test_one_row_of_pages_expanded_to_all_sequences():
    # sequences of different lengths over the same pages, named once
    page, H, kv, hd = 32, 8, 2, 128
    lens, new = [300, 17, 299, 64], [40, 17, 1, 30]
    g = gen(23)
    k, v, table = make_pool(g, [300], page, kv, hd, torch.bfloat16)
    shared, n = i32(table).expand(4, -1), sum(new)
    q = randn(g, n, H, hd, dtype=torch.bfloat16)
    cache, cu = rb.PagedKV(k, v), i32([0, 40, 57, 58, 88])
    check_paged(rb.paged_attention_prompt(cache, rb.PagedBatch(shared, i32(lens), cu, n), q), q, k, v, table * 4, new, lens, hd ** -0.5)
    check_decode(rb.paged_attention_decode(cache, rb.PagedBatch(shared, i32(lens)), q[:4]), q[:4], k, v, table * 4, lens, hd ** -0.5)
    # append: sequences that end at different positions of the pages
    qn, kn, vn = append_inputs(g, 4, H, kv, hd, "bf16", False)
    k0, v0 = k.clone(), v.clone()
    assert torch.equal(rb.paged_append(cache, rb.PagedBatch(shared, i32(lens)), qn, kn, vn), qn)
    for i, m in enumerate(lens):
        at = table[0][(m - 1) // page], (m - 1) % page
        assert torch.equal(k[at], kn[i]) and torch.equal(v[at], vn[i])
        k0[at], v0[at] = kn[i], vn[i]
    assert torch.equal(k, k0) and torch.equal(v, v0)


# ---------------------------------------------------------------- streams
def test_a_batch_dropped_while_its_call_runs():
    # the calls run on a stream that is not current, late; their batch is gone at once and
    # its memory asked for again: the results are right and nobody's memory is written
    lens, H, kv, hd = [4000, 1, 700], 32, 8, 128
    k, v, table, q = decode_case(lens, H, kv, hd, 64, "bf16", False, 6)
    tab, ln, cache = i32(table), i32(lens), rb.PagedKV(k, v)
    want = rb.paged_attention_decode(cache, rb.PagedBatch(tab, ln), q)
    size = rb.lib().rpgc_paged_decode_workspace(cache.ref, len(lens), H)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for how in ("argument", "current", "second stream"):
        batch = rb.PagedBatch(tab, ln)
        if how == "second stream":
            rb.paged_attention_decode(cache, batch, q)
            torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(50_000_000)
            if how == "current":
                got = rb.paged_attention_decode(cache, batch, q)
        if how != "current":
            got = rb.paged_attention_decode(cache, batch, q, stream=side.cuda_stream)
        del batch
        mine = [torch.full((size,), 0xA5, dtype=torch.uint8, device="cuda") for _ in range(8)]
        torch.cuda.synchronize()
        assert torch.equal(got, want), how
        assert all(bool((m == 0xA5).all()) for m in mine), how


def test_one_batch_on_two_streams_at_once():
    lens, H, kv, hd = [3000 + i for i in range(6)], 32, 8, 128
    k, v, table, q = decode_case(lens, H, kv, hd, 64, "bf16", False, 7)
    cache, batch = rb.PagedKV(k, v), rb.PagedBatch(i32(table), i32(lens))
    want = rb.paged_attention_decode(cache, batch, q)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got += [rb.paged_attention_decode(cache, batch, q) for _ in range(5)]
        torch.cuda.synchronize()
        assert all(torch.equal(x, want) for x in got)


# ------------------------------------- values that a row does not see
HUGE = {"bf16": 3.0e38, "f16": 65504.0}  # finite, so that only a weight of zero keeps them out


@pytest.mark.parametrize("lens,H,kv,hd", [([430, 70], 8, 2, 128), ([1500, 300], 32, 8, 128), ([430, 70], 12, 4, 64)])
@pytest.mark.parametrize("ty", ["bf16", "f16"])
def test_large_values_of_later_positions_do_not_leak_into_prompts(lens, H, kv, hd, ty):
    g = gen(sum(lens))
    n, at = sum(lens), 300
    q, k, v = packed_inputs(g, n, H, kv, hd, DT[ty], False)
    cu = i32([0, lens[0], n])
    want = rb.attention_prompt(q, k, v, cu)
    check_packed(want, q, k, v, lens, hd ** -0.5)
    for sign in (1, -1):
        v2 = v.clone()
        v2[at:] = sign * HUGE[ty]
        assert torch.equal(rb.attention_prompt(q, k, v2, cu)[:at], want[:at])


@pytest.mark.parametrize("ty", ["bf16", "f16"])
def test_large_values_past_the_end_do_not_leak_over_pages(ty):
    # later tokens of the prompt, and slots that no sequence holds
    page, H, kv, hd = 32, 8, 2, 128
    g = gen(17)
    lens, new, at = [500, 77], [200, 77], 120  # rows [0, at) see positions below 420
    k, v, table = make_pool(g, lens, page, kv, hd, DT[ty])
    q = randn(g, sum(new), H, hd, dtype=DT[ty])
    cache = rb.PagedKV(k, v)
    batch = rb.PagedBatch(i32(table), i32(lens), i32([0, 200, 277]), 277)
    one = rb.PagedBatch(i32(table), i32(lens))
    want, want1 = rb.paged_attention_prompt(cache, batch, q), rb.paged_attention_decode(cache, one, q[:2])
    used = torch.zeros(k.shape[:2], dtype=torch.bool, device="cuda")
    for s, n in enumerate(lens):
        for j, p in enumerate(table[s]):
            if p >= 0:
                used[p, : max(0, min(page, n - j * page))] = True
    for sign in (1, -1):
        k[~used], v[~used] = sign * HUGE[ty], sign * HUGE[ty]
        assert torch.equal(rb.paged_attention_prompt(cache, batch, q), want)
        assert torch.equal(rb.paged_attention_decode(cache, one, q[:2]), want1)
    for p in range(420, 500):
        v[table[0][p // page], p % page] = HUGE[ty]
    assert torch.equal(rb.paged_attention_prompt(cache, batch, q)[:at], want[:at])


@pytest.mark.parametrize("lens,H,kv,hd", [([430, 70], 8, 2, 128), ([1500, 300], 32, 8, 128), ([430, 70], 12, 4, 64)])
@pytest.mark.parametrize("ty", ["bf16", "f16"])
def test_large_keys_of_later_positions_change_nothing_before_them(lens, H, kv, hd, ty):
    # rows that see them outgrow their references by far; the rows beside them keep
    # theirs, and with them every bit
    g = gen(sum(lens))
    n, at = sum(lens), 300
    q, k, v = packed_inputs(g, n, H, kv, hd, DT[ty], False)
    cu = i32([0, lens[0], n])
    want = rb.attention_prompt(q, k, v, cu)
    for big in (HUGE[ty], -HUGE[ty], 300.0):
        k2 = k.clone()
        k2[at:] = big
        assert torch.equal(rb.attention_prompt(q, k2, v, cu)[:at], want[:at])
    # queries of other rows: each row's result is its own
    q2 = q.clone()
    q2[1::2] *= 64
    assert torch.equal(rb.attention_prompt(q2, k, v, cu)[::2], want[::2])


# -------------------------------------------- infinities that a row sees
def slot(pool, table, s, p):
    return pool[table[s][p // pool.shape[1]], p % pool.shape[1]]


@pytest.mark.parametrize("call", ["paged_attention_decode", "paged_attention_prompt"])
@pytest.mark.parametrize("ty", ["bf16", "f16"])
def test_visible_infinite_values_give_infinities(ty, call):
    # a positive weight times an infinity is that infinity, both signs make NaN;
    # the other dims and the other kv head's rows keep their values
    lens, H, kv, hd = [40, 3000, 5, 700], 8, 2, 128
    k, v, table, q = decode_case(lens, H, kv, hd, 32, ty, False, 3)
    cache, batch = rb.PagedKV(k, v), rb.PagedBatch(i32(table), i32(lens))
    run = getattr(rb, call)
    base, clean = run(cache, batch, q), v.clone()
    for s, n in enumerate(lens):
        a, b = slot(v, table, s, n // 2)[1], slot(v, table, s, n - 1)[1]
        a[3], a[5], a[7], b[7], b[9] = float("inf"), float("-inf"), float("inf"), float("-inf"), float("nan")
    got = run(cache, batch, q)
    assert torch.equal(got[:, :4], base[:, :4])
    assert bool((got[:, 4:, 3] == float("inf")).all()) and bool((got[:, 4:, 5] == float("-inf")).all())
    assert bool(got[:, 4:, [7, 9]].isnan().all())
    got[:, 4:, [3, 5, 7, 9]] = base[:, 4:, [3, 5, 7, 9]]
    check_decode(got, q, k, clean, table, lens, hd ** -0.5)


def ramp_case(scores, ty, hd=128):
    """One sequence whose position t scores scores[t] (scale 1) for the one query head, values of one."""
    n, page = len(scores), 64
    pages = -(-n // page)
    k = torch.zeros(pages, page, 1, hd, dtype=DT[ty], device="cuda")
    k.view(-1, hd)[:n, 0] = torch.tensor(scores, device="cuda").to(DT[ty])
    q = torch.zeros(1, 1, hd, dtype=DT[ty], device="cuda")
    q[0, 0, 0] = 1
    table = [list(range(pages))]
    return k, torch.ones_like(k), table, q


@pytest.mark.parametrize("call", ["paged_attention_decode", "paged_attention_prompt"])
@pytest.mark.parametrize("ty", ["bf16", "f16"])
def test_an_infinite_value_of_little_weight_still_counts(ty, call):
    # e^-40 of the largest weight: nothing in 16 bits, but not zero
    scores = [0.0] * 200
    scores[150] = -40.0
    k, v, table, q = ramp_case(scores, ty)
    v[2, 150 - 128, 0, 6] = float("inf")
    got = getattr(rb, call)(rb.PagedKV(k, v), rb.PagedBatch(i32(table), i32([200])), q, scale=1.0)
    assert float(got[0, 0, 6]) == float("inf")
    got[0, 0, 6] = 1
    assert bool((got == 1).all())


@pytest.mark.parametrize("call", ["paged_attention_decode", "paged_attention_prompt"])
def test_large_values_do_not_overflow_on_the_way(call):
    # the weights outgrow the first keys' by e^22, and the values are 1e30: their
    # products are past fp32's range, the result is not
    scores = ([0.0] * 128 + [22.0] * 128) * 16
    k, v, table, q = ramp_case(scores, "bf16")
    v *= 1e30
    got = getattr(rb, call)(rb.PagedKV(k, v), rb.PagedBatch(i32(table), i32([4096])), q, scale=1.0)
    want = float(v[0, 0, 0, 0])
    assert float((got.double() - want).abs().max()) <= 2.0 ** -8 * want


# ------------------------------------------------- rows of no sequence
@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("norm", [False, True])
def test_append_rows_that_no_sequence_holds_are_zeros(ty, norm):
    # a call of a fixed number of rows, as a captured one is, fewer of them in use:
    # rows before the first sequence, between the bounds' ends and past the last
    page, H, kv, hd, n = 16, 6, 2, 128, 40
    g = gen(11)
    lens, cu = [20, 9, 30], [3, 8, 8, 25]
    k, v, table = make_pool(g, lens, page, kv, hd, torch.bfloat16)
    q, kn, vn = append_inputs(g, n, H, kv, hd, ty, False)
    gain = 1 + 0.1 * randn(g, hd) if norm else None
    tab, status = rb.rope_table(64, hd), i32([0])
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    k0, v0 = k.clone(), v.clone()
    rb.paged_append(rb.PagedKV(k, v), rb.PagedBatch(i32(table), i32(lens), i32(cu), n, status), q, kn, vn, gain, gain, 1e-6, tab,
                    q_out=out)
    assert bool((out[:3] == 0).all()) and bool((out[25:] == 0).all())
    assert bool((out[3:25] != 0).any(-1).all()) and bool((out[3:25] != 7).any(-1).all())
    assert int(status) == 0
    changed = (k != k0).any(-1).any(-1) | (v != v0).any(-1).any(-1)
    assert int(changed.sum()) == 22
    # no sequence at all
    out.fill_(7)
    empty = rb.PagedBatch(i32(table), i32(lens), i32([0, 0, 0, 0]), n, status)
    k0, v0 = k.clone(), v.clone()
    rb.paged_append(rb.PagedKV(k, v), empty, q, kn, vn, gain, gain, 1e-6, tab, q_out=out)
    assert bool((out == 0).all()) and torch.equal(k, k0) and torch.equal(v, v0) and int(status) == 0


# --------------------------------------------------------------- status
def test_calls_without_a_status_word_report_to_the_library():
    g = gen(5)
    k, v, _ = make_pool(g, [64], 16, 2, 64, torch.float16)
    cache, kn = rb.PagedKV(k, v), randn(g, 1, 2, 64)
    rb.paged_status()  # whatever earlier calls left
    rb.paged_append(cache, rb.PagedBatch(i32([[0]]), i32([5])), None, kn, kn)
    rb.paged_attention_decode(cache, rb.PagedBatch(i32([[0]]), i32([5])), kn.half())
    assert rb.paged_status() == 0
    own = i32([0])
    rb.paged_append(cache, rb.PagedBatch(i32([[-1]]), i32([5]), status=own), None, kn, kn)
    assert rb.paged_status() == 0 and int(own) == rb.paged.DROPPED
    rb.paged_append(cache, rb.PagedBatch(i32([[-1]]), i32([5])), None, kn, kn)
    assert rb.paged_status() == rb.paged.DROPPED
    assert rb.paged_status() == 0  # told once


# ------------------------------------------------------------- precision
@pytest.mark.parametrize("ty", ["bf16", "f16"])
@pytest.mark.parametrize("n", [96, 4000])
def test_decode_weights_keep_more_than_16_bits(ty, n):
    # Weights that round to 16 bits as badly as they can, values that cancel.  Every 16
    # positions have two of score 0 and value 0, the reference of whoever takes those 16; of
    # the others, one half weigh a little less than halfway above a 16-bit number in [1/2, 1)
    # and hold 1, the other half a little more than halfway above another and hold -1.
    # Bound: the output's rounding, u / 2 of the value, and 2^-13 of sum p |v| for
    # everything before it (weights in two 16-bit parts are within 2^-17; ex2 and its
    # fp32 argument, at most 1 here, 2^-22; fp32 sums of up to 4000 / 16 steps 2^-15).
    # Weights of one 16-bit part err by 0.48 steps of 2^-8 (bf16) or 2^-11 (fp16) of
    # 1/2, with the values all in one direction: 2^-8 or 2^-11 of sum p |v|, which is above
    # the bound.
    dt, hd, page, step = DT[ty], 64, 32, 2.0 ** (-8 if ty == "bf16" else -11)
    kind = torch.tensor([0 if i % 16 in (0, 15) else 1 + i % 2 for i in range(n)], device="cuda")
    s = torch.tensor([0.0, np.log(0.5 + 0.48 * step), np.log(0.5 + 7.52 * step)], dtype=torch.float64, device="cuda")
    parts, rest = [], s.clone()
    for _ in range(4):  # exact in a few 16-bit parts, each times 1 of q
        parts.append(rest.to(dt))
        rest = rest - parts[-1].double()
    s = sum(p.double() for p in parts)  # what the scores are
    pages = -(-n // page)
    k = torch.zeros(pages, page, 1, hd, dtype=dt, device="cuda")
    v = torch.zeros_like(k)
    for i, p in enumerate(parts):
        k.view(-1, hd)[:n, i] = p[kind]
    w = torch.exp(s)[kind]
    vals = torch.tensor([0.0, 1.0, -1.0], dtype=torch.float64, device="cuda")[kind].to(dt)
    v.view(-1, hd)[:n] = vals[:, None]
    q = torch.zeros(1, 1, hd, dtype=dt, device="cuda")
    q[..., :4] = 1
    got = rb.paged_attention_decode(rb.PagedKV(k, v), rb.PagedBatch(i32([list(range(pages))]), i32([n])), q, scale=1.0)
    e, mag = (w * vals.double()).sum() / w.sum(), (w * vals.double().abs()).sum() / w.sum()
    bound = float(U[dt] / 2 * e.abs() + 2.0 ** -13 * mag)
    assert float((got.double() - e).abs().max()) <= bound
    once = ((w.to(dt).double() * vals.double()).sum() / w.sum() - e).abs()
    assert float(once) > (3 if ty == "f16" else 15) * bound  # weights rounded to 16 bits would be seen


# ------------------------------------------------- bounds that make no sense
@pytest.mark.parametrize("cu", [[-5, 100, 40, 9999], [300, 200, 100, 0], [0, 2 ** 31 - 1, -2 ** 31, 300], [299, 299, 300, 300]])
def test_prompt_bounds_out_of_range_write_inside_the_result(cu):
    # bounds that leave [0, n_tokens] or fall are kept inside it; nothing beside `out` is
    # written, no wait gives up, rows of sequences whose bounds are in order are right
    g = gen(31)
    n, H, kv, hd, page = 300, 4, 2, 64, 32
    q, k, v = packed_inputs(g, n, H, kv, hd, torch.float16, False)
    guard = 64 * H * hd
    buf = torch.full((n * H * hd + 2 * guard,), 3.0, dtype=torch.float16, device="cuda")
    out, status = buf[guard:-guard].view(n, H, hd), i32([0])
    rb.attention_prompt(q, k, v, i32(cu), out=out, status=status)
    assert int(status) == 0
    assert bool((buf[:guard] == 3).all()) and bool((buf[-guard:] == 3).all())
    assert torch.isfinite(out).all()
    bounds = [min(max(c, 0), n) for c in cu]
    held = torch.zeros(n, dtype=torch.int32)
    for a, b in zip(bounds, bounds[1:]):
        held[a:b] += 1
    assert bool((out[(held == 0).cuda()] == 3).all())
    for a, b in zip(bounds, bounds[1:]):
        if b > a and int(held[a:b].max()) == 1:
            check_packed(out[a:b], q[a:b], k[a:b], v[a:b], [b - a], hd ** -0.5)
    # over pages: the same bounds, more new rows than positions among them
    kp, vp, table = make_pool(g, [n, n, n], page, kv, hd, torch.float16)
    buf.fill_(3)
    rb.paged_attention_prompt(rb.PagedKV(kp, vp), rb.PagedBatch(i32(table), i32([n, 5, n]), i32(cu), n, status), q, out=out)
    assert int(status) == 0
    assert bool((buf[:guard] == 3).all()) and bool((buf[-guard:] == 3).all())
    assert torch.isfinite(out).all() and bool((out[(held == 0).cuda()] == 3).all())


# ---------------------------------------------------------- broadcast inputs
def test_heads_and_rows_expanded_from_one():
    # strides of zero: one K and V head read as four, one query row as all
    g = gen(41)
    n, H, hd, page = 150, 8, 128, 16
    q, k1, v1 = randn(g, 1, H, hd, dtype=torch.bfloat16), randn(g, n, 1, hd, dtype=torch.bfloat16), randn(g, n, 1, hd, dtype=torch.bfloat16)
    q, k, v = q.expand(n, -1, -1), k1.expand(-1, 4, -1), v1.expand(-1, 4, -1)
    cu = i32([0, 100, n])
    assert torch.equal(rb.attention_prompt(q, k, v, cu), rb.attention_prompt(*(x.contiguous() for x in (q, k, v)), cu))
    kp, vp, table = make_pool(g, [90, 150], page, 1, hd, torch.bfloat16)
    wide, full = rb.PagedKV(kp.expand(-1, -1, 4, -1), vp.expand(-1, -1, 4, -1)), rb.PagedKV(kp.repeat(1, 1, 4, 1), vp.repeat(1, 1, 4, 1))
    batch = rb.PagedBatch(i32(table), i32([90, 150]))
    assert torch.equal(rb.paged_attention_decode(wide, batch, q[:2]), rb.paged_attention_decode(full, batch, q[:2].contiguous()))
    batch = rb.PagedBatch(i32(table), i32([90, 150]), i32([0, 30, 100]), 100)
    assert torch.equal(rb.paged_attention_prompt(wide, batch, q[:100]), rb.paged_attention_prompt(full, batch, q[:100].contiguous()))
    # append of one row to every sequence
    qa, ka = randn(g, 1, H, hd).expand(2, -1, -1), randn(g, 1, 1, hd).expand(2, 1, -1)
    one, both = rb.PagedKV(kp.clone(), vp.clone()), rb.PagedKV(kp.clone(), vp.clone())
    batch = rb.PagedBatch(i32(table), i32([90, 150]))
    assert torch.equal(rb.paged_append(one, batch, qa, ka, ka), rb.paged_append(both, batch, qa.contiguous(), ka.contiguous(), ka.contiguous()))
    assert torch.equal(one.k, both.k) and torch.equal(one.v, both.v)
