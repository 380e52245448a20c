"""Argument checks of the paged-cache entry points through the C ABI: they run
before any device work, so no GPU is needed (no pointer is followed)."""
import ctypes as C

import pytest

import rpgbarengine_b200 as rb
from rpgbarengine_b200 import paged

P = 1 << 20  # a 16-byte aligned address that nothing reads


def kv(**kw):
    c = paged._KV(P, P, (C.c_int64 * 3)(16 * 8 * 128, 8 * 128, 128), (C.c_int64 * 3)(16 * 8 * 128, 8 * 128, 128),
                  rb.F16, 10, 16, 8, 128)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def batch(**kw):
    b = paged._Batch(P, 4, 4, 2, P, None, 2, None)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def decode(c=None, b=None, q=P, st=(1024, 128), heads=16, scale=0.1, out=P, ws=P, ws_bytes=1 << 40):
    return rb.lib().rpgc_paged_attention_decode(
        None if c is False else C.byref(c or kv()), None if b is False else C.byref(b or batch()), q,
        (C.c_int64 * 2)(*st) if st else None, heads, scale, out, ws, ws_bytes, None)


def says(rc, word):
    assert rc == rb.E_ARG
    assert word in rb.lib().rpgc_last_error().decode(), rb.lib().rpgc_last_error()


S3 = C.c_int64 * 3


@pytest.mark.parametrize("kw,word", [
    (dict(k=None), "kv->k"), (dict(v=None), "kv->v"), (dict(k=P + 8), "aligned"), (dict(type=rb.F32), "type"),
    (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"), (dict(page_size=512), "page_size"),
    (dict(n_pages=0), "n_pages"), (dict(n_kv_heads=0), "n_kv_heads"), (dict(head_dim=96), "head_dim"),
    (dict(k_stride=S3(100, 4, 128)), "stride"), (dict(v_stride=S3(-8, 8, 8)), "stride"),
    (dict(n_kv_heads=3), "n_heads"), (dict(n_kv_heads=32), "n_heads"),
])
def test_cache_is_checked(kw, word):
    says(decode(kv(**kw)), word)


@pytest.mark.parametrize("kw,word", [
    (dict(block_table=None), "block_table"), (dict(kv_lens=None), "kv_lens"), (dict(max_pages=0), "max_pages"),
    (dict(table_stride=3), "table_stride"), (dict(n_seqs=-1), "n_seqs"), (dict(n_tokens=3), "one token per sequence"),
    (dict(block_table=P + 2), "block_table"), (dict(kv_lens=P + 1), "kv_lens"), (dict(status=P + 2), "status"),
    (dict(n_tokens=-1), "n_tokens"), (dict(n_tokens=1 << 25), "n_tokens"), (dict(cu_q=P), "cu_q"),
])
def test_batch_is_checked(kw, word):
    says(decode(b=batch(**kw)), word)


@pytest.mark.parametrize("kw,word", [
    (dict(c=False), "kv is NULL"), (dict(b=False), "batch is NULL"), (dict(q=None), "q is NULL"), (dict(out=None), "out is NULL"),
    (dict(out=P + 2), "aligned"), (dict(st=None), "q_stride"), (dict(st=(4, 128)), "stride"), (dict(heads=12), "n_heads"),
    (dict(heads=17 * 8), "n_heads"), (dict(heads=0), "n_heads"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(ws=None), "workspace"),
    (dict(ws_bytes=0), "workspace"),
])
def test_decode_call_is_checked(kw, word):
    says(decode(**kw), word)


def test_workspace_size_is_checked():
    L = rb.lib()
    assert L.rpgc_paged_decode_workspace(C.byref(kv()), 4, 16) > 0
    says(L.rpgc_paged_decode_workspace(None, 4, 16), "kv is NULL")
    says(L.rpgc_paged_decode_workspace(C.byref(kv()), -1, 16), "n_seqs")
    says(L.rpgc_paged_decode_workspace(C.byref(kv()), 4, 15), "n_heads")


def append(c=None, b=None, ty=rb.F32, q=P, heads=16, k=P, v=P, st=(1024, 128), qn=P, kn=P, eps=1e-6, rope=P, rows=8, qo=P):
    s = (C.c_int64 * 2)(*st) if st else None
    return rb.lib().rpgc_paged_append(C.byref(c or kv()), C.byref(b or batch()), ty, q, s, heads, k, s, v, s, qn, kn, eps,
                                      rope, rows, qo, None)


@pytest.mark.parametrize("kw,word", [
    (dict(ty=rb.Q8_0), "type"), (dict(q=None), "together"), (dict(qo=None), "together"), (dict(kn=None), "together"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(rows=0), "rope_rows"), (dict(k=None), "k is NULL"),
    (dict(v=P + 4), "aligned"), (dict(st=None), "strides"), (dict(st=(1024, 2)), "stride"), (dict(heads=4), "n_heads"),
    (dict(rope=P + 4), "aligned"), (dict(qn=P + 4), "aligned"),
])
def test_append_call_is_checked(kw, word):
    says(append(**kw), word)


def packed(ty=rb.BF16, q=P, k=P, v=P, st=(1024, 128), cu=P, n_seqs=1, n=4, heads=8, kvh=8, hd=128, scale=0.1, out=P):
    s = (C.c_int64 * 2)(*st) if st else None
    return rb.lib().rpgc_attention_prompt(ty, q, s, k, s, v, s, cu, n_seqs, n, heads, kvh, hd, scale, out, None, None)


@pytest.mark.parametrize("kw,word", [
    (dict(ty=rb.F32), "type"), (dict(q=None), "q is NULL"), (dict(k=None), "k is NULL"), (dict(v=None), "v is NULL"),
    (dict(cu=None), "cu is NULL"), (dict(st=None), "stride"), (dict(st=(1020, 128)), "stride"), (dict(n_seqs=-1), "n_seqs"),
    (dict(n=-1), "n_tokens"), (dict(heads=9), "n_heads"), (dict(hd=80), "head_dim"), (dict(scale=-0.5), "scale"),
    (dict(out=P + 1), "aligned"),
])
def test_packed_call_is_checked(kw, word):
    says(packed(**kw), word)


def test_empty_calls_do_nothing():
    # nothing to do is not an error, and launches nothing
    before = rb.kernel_launches()
    assert packed(n_seqs=0) == rb.OK and packed(n=0) == rb.OK
    assert decode(b=batch(n_seqs=0, n_tokens=0)) == rb.OK
    assert append(b=batch(n_seqs=0, n_tokens=0)) == rb.OK
    assert rb.kernel_launches() == before
