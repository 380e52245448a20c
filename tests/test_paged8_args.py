"""Argument checks of the 8-bit paged cache's and the shared prefixes' entry points
through the C ABI: they run before any device work, so no GPU is needed (no pointer is
followed)."""
import ctypes as C

import pytest

import rpgbarengine_b200 as rb
from rpgbarengine_b200 import paged

P = 1 << 20  # a 16-byte aligned address that nothing reads
S3 = C.c_int64 * 3


def fields(c, kw):
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def kv8(**kw):
    return fields(paged._KV8(P, P, S3(16 * 8 * 128, 8 * 128, 128), S3(16 * 8 * 128, 8 * 128, 128), P, paged._S2(256, 32), rb.F16, 10, 16, 8, 128), kw)


def kv(**kw):
    return fields(paged._KV(P, P, S3(16 * 8 * 128, 8 * 128, 128), S3(16 * 8 * 128, 8 * 128, 128), rb.F16, 10, 16, 8, 128), kw)


def batch(**kw):
    return fields(paged._Batch(P, 4, 4, 2, P, None, 2, None), kw)


def prefix(cache=None, **kw):
    cache = cache or kv()
    p = fields(paged._Prefix(C.pointer(cache), P, 4, 4, 1, P, P), kw)
    p.held = cache
    return p


def decode(c=None, b=None, pre=None, q=P, st=(1024, 128), heads=16, scale=0.1, out=P, ws=P, ws_bytes=1 << 40, fn="rpgc_paged8_attention_decode"):
    return getattr(rb.lib(), fn)(None if c is False else C.byref(c or (kv8() if "8" in fn else kv())), C.byref(b or batch()),
                                 None if pre is None else C.byref(pre), q, (C.c_int64 * 2)(*st) if st else None, heads, scale, out, ws, ws_bytes, None)


def says(rc, word):
    assert rc == rb.E_ARG
    assert word in rb.lib().rpgc_last_error().decode(), rb.lib().rpgc_last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(k=None), "kv->k"), (dict(v=None), "kv->v"), (dict(k=P + 8), "aligned"), (dict(type=rb.F32), "type"),
    (dict(page_size=8), "page_size"), (dict(n_pages=0), "n_pages"), (dict(n_kv_heads=0), "n_kv_heads"), (dict(head_dim=96), "head_dim"),
    (dict(k_stride=S3(100, 8, 128)), "stride"), (dict(v_stride=S3(-16, 16, 16)), "stride"), (dict(k_stride=S3(16384, 1024, 8)), "stride"),
    (dict(scales=None), "scales"), (dict(scales=P + 4), "scales"), (dict(scale_stride=paged._S2(256, 30)), "stride"),
    (dict(scale_stride=paged._S2(-4, 32)), "stride"), (dict(n_kv_heads=3), "n_heads"),
])
def test_cache_is_checked(kw, word):
    says(decode(kv8(**kw)), word)
    if "n_heads" not in word:
        says(append(kv8(**kw)), word)
        says(read(kv8(**kw)), word)


@pytest.mark.parametrize("fn", ["rpgc_paged8_attention_decode", "rpgc_paged_attention_decode_prefix"])
@pytest.mark.parametrize("kw,word", [
    (dict(c=False), "kv is NULL"), (dict(q=None), "q is NULL"), (dict(out=None), "out is NULL"), (dict(out=P + 2), "aligned"),
    (dict(st=None), "q_stride"), (dict(st=(4, 128)), "stride"), (dict(heads=12), "n_heads"), (dict(heads=17 * 8), "n_heads"),
    (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(ws=None), "workspace"), (dict(ws_bytes=0), "workspace"),
    (dict(b=batch(cu_q=P)), "cu_q"), (dict(b=batch(kv_lens=None)), "kv_lens"), (dict(b=batch(n_tokens=3)), "one token per sequence"),
])
def test_decode_call_is_checked(fn, kw, word):
    says(decode(**{"pre": prefix(), "fn": fn, **kw}), word)


@pytest.mark.parametrize("fn", ["rpgc_paged8_attention_decode", "rpgc_paged_attention_decode_prefix"])
@pytest.mark.parametrize("cache,kw,word", [
    (kv(k=None), {}, "kv->k"), (kv(n_kv_heads=4), {}, "prefix"), (kv(head_dim=64), {}, "prefix"), (kv(type=rb.BF16), {}, "prefix"),
    (kv(), dict(block_table=None), "block_table"), (kv(), dict(lens=None), "lens"), (kv(), dict(cu_seqs=None), "cu_seqs"),
    (kv(), dict(block_table=P + 1), "block_table"), (kv(), dict(lens=P + 2), "lens"), (kv(), dict(cu_seqs=P + 3), "cu_seqs"),
    (kv(), dict(n_groups=-1), "n_groups"), (kv(), dict(max_pages=0), "max_pages"), (kv(), dict(table_stride=2), "table_stride"),
])
def test_prefix_is_checked(fn, cache, kw, word):
    says(decode(pre=prefix(cache, **kw), fn=fn), word)


def test_a_prefix_call_needs_one():
    says(decode(fn="rpgc_paged_attention_decode_prefix"), "prefix is NULL")


def test_workspace_sizes_are_checked():
    L = rb.lib()
    assert L.rpgc_paged8_decode_workspace(C.byref(kv8()), 4, 16) > 0
    assert L.rpgc_paged_prefix_workspace(4, 16, 8, 128) > 0
    says(L.rpgc_paged8_decode_workspace(None, 4, 16), "kv is NULL")
    says(L.rpgc_paged8_decode_workspace(C.byref(kv8()), -1, 16), "n_seqs")
    says(L.rpgc_paged_prefix_workspace(4, 15, 8, 128), "n_heads")
    says(L.rpgc_paged_prefix_workspace(4, 16, 8, 100), "head_dim")
    says(L.rpgc_paged_prefix_workspace(-1, 16, 8, 128), "n_seqs")


def append(c=None, b=None, ty=rb.F32, q=P, heads=16, k=P, v=P, st=(1024, 128), qn=P, kn=P, eps=1e-6, rope=P, rows=8, qo=P):
    s = (C.c_int64 * 2)(*st) if st else None
    return rb.lib().rpgc_paged8_append(C.byref(c or kv8()), C.byref(b or batch()), ty, q, s, heads, k, s, v, s, qn, kn, eps, rope, rows, qo, None)


@pytest.mark.parametrize("kw,word", [
    (dict(ty=rb.Q8_0), "type"), (dict(q=None), "together"), (dict(kn=None), "together"), (dict(eps=-1.0), "eps"), (dict(rows=0), "rope_rows"),
    (dict(k=None), "k is NULL"), (dict(v=P + 4), "aligned"), (dict(st=None), "strides"), (dict(st=(1024, 2)), "stride"), (dict(heads=4), "n_heads"),
])
def test_append_call_is_checked(kw, word):
    says(append(**kw), word)


def read(c=None, b=None, to=None, tab=P, stride=4, pages=4):
    return rb.lib().rpgc_paged8_read(C.byref(c or kv8()), C.byref(b or batch()), None if to is False else C.byref(to or kv()), tab, stride, pages, None)


@pytest.mark.parametrize("kw,word", [
    (dict(to=False), "kv is NULL"), (dict(to=kv(n_kv_heads=4)), "to's"), (dict(to=kv(head_dim=64)), "to's"), (dict(tab=None), "to_table"),
    (dict(tab=P + 2), "to_table"), (dict(pages=0), "max_pages"), (dict(stride=2), "table_stride"), (dict(b=batch(block_table=None)), "block_table"),
])
def test_read_call_is_checked(kw, word):
    says(read(**kw), word)


def test_empty_calls_do_nothing():
    before, none = rb.kernel_launches(), batch(n_seqs=0, n_tokens=0)
    assert decode(b=none) == rb.OK and append(b=none) == rb.OK and read(b=none) == rb.OK
    assert decode(b=none, pre=prefix(), fn="rpgc_paged_attention_decode_prefix") == rb.OK
    assert rb.kernel_launches() == before


# ------------------------------------------------------- the Python layer
torch = pytest.importorskip("torch")


class Dev:
    """A CPU tensor that says it is on CUDA device 0."""
    is_cuda = True

    def __init__(self, t):
        self.t = t

    def get_device(self):
        return 0

    def __getattr__(self, name):
        return getattr(self.t, name)


def ints(v):
    return Dev(torch.tensor(v, dtype=torch.int32))


def pool(dtype=torch.float8_e4m3fn, shape=(3, 16, 2, 64)):
    return Dev(torch.zeros(shape).to(dtype))


def refused(word, fn, *args, **kw):
    with pytest.raises(rb.RpgcError) as e:
        fn(*args, **kw)
    assert e.value.code == rb.E_ARG and word in str(e.value)


def test_a_cache_of_8_bits_says_where_its_scales_are():
    s = torch.zeros(3, 2, 2, 16)
    c = rb.PagedKV8(pool(), pool(), Dev(s)).c
    assert list(c.scale_stride) == [64, 32] and list(c.k_stride) == [16 * 128, 128, 64] and c.type == rb.BF16
    wide = torch.zeros(3, 5, 3, 16)[:, 1:3, :2]
    assert list(rb.PagedKV8(pool(), pool(), Dev(wide), dtype=torch.float16).c.scale_stride) == [240, 48]


def test_pools_are_checked():
    s = Dev(torch.zeros(3, 2, 2, 16))
    refused("float8_e4m3fn", rb.PagedKV8, pool(torch.float16), pool(torch.float16), s)
    refused("one shape", rb.PagedKV8, pool(), pool(shape=(3, 16, 2, 128)), s)
    refused("scales", rb.PagedKV8, pool(), pool(), Dev(torch.zeros(3, 16, 2, 2)))
    refused("scales", rb.PagedKV8, pool(), pool(), Dev(torch.zeros(3, 2, 2, 16, dtype=torch.float64)))
    refused("scales", rb.PagedKV8, pool(), pool(), Dev(torch.zeros(3, 2, 16, 2).transpose(2, 3)))
    refused("dtype", rb.PagedKV8, pool(), pool(), s, dtype=torch.float32)


def test_prefixes_are_checked():
    c16 = rb.PagedKV(pool(torch.float16), pool(torch.float16))
    c8 = rb.PagedKV8(pool(), pool(), Dev(torch.zeros(3, 2, 2, 16)), dtype=torch.float16)
    ok = rb.PagedPrefix(c16, ints([[0, 1]]), ints([20]), ints([0, 2]))
    assert ok.c.table_stride == 2 and ok.c.n_groups == 1
    wide = Dev(torch.zeros(2, 6, dtype=torch.int32)[:, :2])
    assert rb.PagedPrefix(c16, wide, ints([20, 3]), ints([0, 2, 2])).c.table_stride == 6
    refused("16 bits", rb.PagedPrefix, c8, ints([[0, 1]]), ints([20]), ints([0, 2]))
    refused("cu_seqs", rb.PagedPrefix, c16, ints([[0, 1]]), ints([20]), ints([0, 2, 3]))
    refused("block_table", rb.PagedPrefix, c16, ints([[0, 1]]), ints([20, 30]), ints([0, 2, 3]))
    refused("int32", rb.PagedPrefix, c16, ints([[0, 1]]), Dev(torch.zeros(1)), ints([0, 2]))
    refused("lens", rb.PagedPrefix, c16, ints([[0, 1]] * 2), Dev(torch.zeros(4, dtype=torch.int32)[::2]), ints([0, 1, 2]))


def test_calls_on_the_wrong_cache_are_refused():
    c16 = rb.PagedKV(pool(torch.float16), pool(torch.float16))
    c8 = rb.PagedKV8(pool(), pool(), Dev(torch.zeros(3, 2, 2, 16)), dtype=torch.float16)
    b = rb.PagedBatch(ints([[0]]), ints([3]))
    q = Dev(torch.zeros(1, 4, 64, dtype=torch.float16))
    refused("paged_read", rb.paged_attention_prompt, c8, rb.PagedBatch(ints([[0]]), ints([3]), ints([0, 1]), 1), q)
    refused("PagedKV8", rb.paged_read, c16, b, c16, ints([[0]]))
    refused("PagedKV8", rb.paged_read, c8, b, c8, ints([[0]]))
    refused("to_table", rb.paged_read, c8, b, c16, ints([[0], [1]]))
    refused("type", rb.paged_attention_decode, c8, b, Dev(torch.zeros(1, 4, 64, dtype=torch.bfloat16)))
