"""Paged KV cache on the device (rpgc_paged_*, rpgc_attention_prompt).

  PagedKV                  one layer's K and V pools: [page, position, kv head, head_dim]
  PagedBatch               the sequences of a call: block table, lengths, packed rows
  paged_append             QK-norm + RoPE + write of new tokens into their pages
  paged_attention_decode   one new token per sequence over its pages
  paged_attention_prompt   causal attention of packed prompts over their pages
  attention_prompt         the same with K and V packed beside q
  rope_table               the cosine and sine rows paged_append reads

Lengths, tables and page ids live on the device and are read there when the
call runs: nothing here waits for the GPU, and all calls can be captured.
"""
from __future__ import annotations

import ctypes as C
import math

from . import BF16, E_ARG, F16, F32, RpgcError, _check, lib

DROPPED, TIMEOUT = 1, 2  # PagedBatch.status bits


class _KV(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_stride", C.c_int64 * 3), ("v_stride", C.c_int64 * 3),
                ("type", C.c_uint32), ("n_pages", C.c_int32), ("page_size", C.c_int32),
                ("n_kv_heads", C.c_int32), ("head_dim", C.c_int32)]


class _Batch(C.Structure):
    _fields_ = [("block_table", C.c_void_p), ("table_stride", C.c_int64), ("max_pages", C.c_int32),
                ("n_seqs", C.c_int32), ("kv_lens", C.c_void_p), ("cu_q", C.c_void_p),
                ("n_tokens", C.c_int64), ("status", C.c_void_p)]


_S2 = C.c_int64 * 2


def _need(ok, msg):
    if not ok:
        raise RpgcError(E_ARG, msg)


def _type(t):
    import torch
    ty = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}.get(t.dtype)
    _need(ty is not None, f"{t.dtype} is not supported")
    return ty


def _ints(t, what, dims):
    import torch
    _need(t.is_cuda and t.dtype == torch.int32 and t.dim() == dims, f"{what} must be a {dims}-D int32 CUDA tensor")


def _rows(t, what, dev, shape):
    """Strides of a [token, head, dim] tensor with contiguous rows on `dev`."""
    _need(t.device == dev and t.dim() == 3, f"{what} must be a 3-D tensor on {dev}")
    _need(all(a == b for a, b in zip(t.shape, shape) if b is not None), f"{what} has shape {tuple(t.shape)}")
    s = t.stride()
    _need(s[2] == 1, f"{what}: rows of head_dim values must be contiguous")
    return _S2(s[0], s[1])


def _result(out, shape, dtype, dev, what):
    import torch
    if out is None:
        return torch.empty(shape, dtype=dtype, device=dev)
    _need(out.device == dev and out.dtype == dtype and tuple(out.shape) == tuple(shape) and out.is_contiguous(),
          f"{what} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {dev}")
    return out


class _On:
    """The stream a call runs on, with its device current."""

    def __init__(self, dev, stream):
        import torch
        self.cuda = torch.cuda
        self.guard = torch.cuda.device(dev) if dev.index != torch.cuda.current_device() else None
        self.other = stream
        self.ptr = int(torch.cuda.current_stream(dev).cuda_stream if stream is None else stream)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return self

    def __exit__(self, *e):
        if self.guard is not None:
            self.guard.__exit__(*e)

    def keep(self, t):
        """A result made here on the current stream and used on another one
        keeps its memory until that stream is done with it."""
        if self.other is not None:
            t.record_stream(self.cuda.ExternalStream(self.ptr, device=t.device))


class PagedKV:
    """One layer's K and V pools, [n_pages, page_size, n_kv_heads, head_dim]
    in float16 or bfloat16, any strides that are multiples of 8 elements (a
    head-major pool is passed transposed).  Holds references to both."""

    def __init__(self, k, v):
        _need(k.is_cuda and k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype and k.device == v.device,
              "k and v must be 4-D CUDA tensors of one shape and type")
        _need(k.stride(3) == 1 and v.stride(3) == 1, "rows of head_dim values must be contiguous")
        self.k, self.v, self.device, self.dtype = k, v, k.device, k.dtype
        n, p, h, d = k.shape
        ty = _type(k)
        _need(ty != F32, "a paged cache holds float16 or bfloat16")
        self.c = _KV(k.data_ptr(), v.data_ptr(), (C.c_int64 * 3)(*k.stride()[:3]), (C.c_int64 * 3)(*v.stride()[:3]),
                     ty, n, p, h, d)
        self.ref = C.byref(self.c)
        self.page_size, self.n_kv_heads, self.head_dim = p, h, d

    @classmethod
    def empty(cls, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, dtype=None, device="cuda") -> "PagedKV":
        """New pools (bfloat16 unless said otherwise); their values are never
        read before append writes them."""
        import torch
        shape, dt = (n_pages, page_size, n_kv_heads, head_dim), dtype or torch.bfloat16
        return cls(torch.empty(shape, dtype=dt, device=device), torch.empty(shape, dtype=dt, device=device))


class PagedBatch:
    """The sequences of a call.  block_table: int32 [n_seqs, max_pages] page
    ids; kv_lens: int32 [n_seqs] cache lengths, the call's new tokens included;
    cu_q: int32 [n_seqs + 1], sequence s's new tokens are rows
    [cu_q[s], cu_q[s+1]) of n_tokens (None: one new token per sequence).  All on
    the device, and read there at each call, so a decode loop updates them in
    place and keeps the batch.  status: optional int32 tensor of one word that
    receives DROPPED / TIMEOUT bits.  The batch also holds decode's workspace:
    calls on one batch are made in stream order."""

    def __init__(self, block_table, kv_lens, cu_q=None, n_tokens=None, status=None):
        _ints(block_table, "block_table", 2)
        _ints(kv_lens, "kv_lens", 1)
        n = kv_lens.shape[0]
        _need(block_table.shape[0] == n and block_table.stride(1) == 1, "block_table needs one contiguous row per sequence")
        _need(kv_lens.stride(0) == 1 or n < 2, "kv_lens must be contiguous")
        if cu_q is not None:
            _ints(cu_q, "cu_q", 1)
            _need(cu_q.shape[0] == n + 1 and cu_q.stride(0) == 1, "cu_q must hold n_seqs + 1 contiguous values")
            _need(n_tokens is not None, "n_tokens is needed with cu_q")
        if status is not None:
            _ints(status, "status", 1)
        self.keep = (block_table, kv_lens, cu_q, status)
        self.device = kv_lens.device
        _need(all(t is None or t.device == self.device for t in self.keep), "the batch's tensors must be on one device")
        self.n_seqs, self.n_tokens = n, n if n_tokens is None else int(n_tokens)
        p = [None if t is None else t.data_ptr() for t in self.keep]
        self.c = _Batch(p[0], max(block_table.stride(0), block_table.shape[1]), block_table.shape[1], n, p[1], p[2],
                        self.n_tokens, p[3])
        self.ref = C.byref(self.c)
        self._ws = {}

    def workspace(self, cache: PagedKV, n_heads: int):
        """Decode's workspace for this batch and head count (made once)."""
        key = (n_heads, cache.n_kv_heads, cache.head_dim)
        ws = self._ws.get(key)
        if ws is None:
            import torch
            n = _check(lib().rpgc_paged_decode_workspace(cache.ref, self.n_seqs, n_heads))
            ws = self._ws[key] = torch.zeros(n, dtype=torch.uint8, device=self.device)
        return ws


def paged_append(cache: PagedKV, batch: PagedBatch, q, k, v, q_norm=None, k_norm=None, eps: float = 1e-6, rope=None,
                 q_out=None, stream=None):
    """Writes the batch's new tokens into their pages and returns q normalised
    and rotated in the cache's type (None when q is None).  q [n_tokens,
    n_heads, head_dim], k and v [n_tokens, n_kv_heads, head_dim], of one type
    (float32, float16 or bfloat16); q_norm / k_norm: fp32 gains [head_dim] or
    None; rope: fp32 [positions, head_dim] (rope_table) or None."""
    import torch
    dev, n, d = cache.device, batch.n_tokens, cache.head_dim
    _need(batch.device == dev, "cache and batch are on different devices")
    ty = _type(k)
    _need(v.dtype == k.dtype and (q is None or q.dtype == k.dtype), "q, k and v must have one type")
    ks = _rows(k, "k", dev, (n, cache.n_kv_heads, d))
    vs = _rows(v, "v", dev, (n, cache.n_kv_heads, d))
    qs = None if q is None else _rows(q, "q", dev, (n, None, d))
    for g in (q_norm, k_norm):
        _need(g is None or (g.device == dev and g.dtype == torch.float32 and g.shape == (d,) and (g.stride(0) == 1)),
              "norm gains must be contiguous float32 [head_dim]")
    _need(rope is None or (rope.device == dev and rope.dtype == torch.float32 and rope.dim() == 2 and
                           rope.shape[1] == d and rope.is_contiguous()), "rope must be contiguous float32 [positions, head_dim]")
    heads = 0 if q is None else q.shape[1]
    with _On(dev, stream) as on:
        made = q is not None and q_out is None
        q_out = None if q is None else _result(q_out, (n, heads, d), cache.dtype, dev, "q_out")
        _check(lib().rpgc_paged_append(
            cache.ref, batch.ref, ty, None if q is None else q.data_ptr(), qs, heads, k.data_ptr(), ks, v.data_ptr(), vs,
            None if q_norm is None else q_norm.data_ptr(), None if k_norm is None else k_norm.data_ptr(), eps,
            None if rope is None else rope.data_ptr(), 0 if rope is None else rope.shape[0],
            None if q is None else q_out.data_ptr(), on.ptr))
        if made:
            on.keep(q_out)
    return q_out


def paged_attention_decode(cache: PagedKV, batch: PagedBatch, q, scale=None, out=None, stream=None):
    """Attention of one new token per sequence, q [n_seqs, n_heads, head_dim],
    over the sequence's positions; returns the same shape.  scale: default
    head_dim ** -0.5."""
    dev, d = cache.device, cache.head_dim
    _need(batch.device == dev and q.dtype == cache.dtype, "q, cache and batch must share their device, q the cache's type")
    qs = _rows(q, "q", dev, (batch.n_tokens, None, d))
    heads = q.shape[1]
    with _On(dev, stream) as on:
        made = out is None
        out = _result(out, q.shape, cache.dtype, dev, "out")
        ws = batch.workspace(cache, heads)
        _check(lib().rpgc_paged_attention_decode(cache.ref, batch.ref, q.data_ptr(), qs, heads,
                                                 d ** -0.5 if scale is None else scale, out.data_ptr(), ws.data_ptr(),
                                                 ws.numel(), on.ptr))
        if made:
            on.keep(out)
    return out


def paged_attention_prompt(cache: PagedKV, batch: PagedBatch, q, scale=None, out=None, stream=None):
    """Causal attention of the batch's new tokens, q [n_tokens, n_heads,
    head_dim], over their sequences' pages (a cached prefix included)."""
    dev, d = cache.device, cache.head_dim
    _need(batch.device == dev and q.dtype == cache.dtype, "q, cache and batch must share their device, q the cache's type")
    qs = _rows(q, "q", dev, (batch.n_tokens, None, d))
    with _On(dev, stream) as on:
        made = out is None
        out = _result(out, q.shape, cache.dtype, dev, "out")
        _check(lib().rpgc_paged_attention_prompt(cache.ref, batch.ref, q.data_ptr(), qs, q.shape[1],
                                                 d ** -0.5 if scale is None else scale, out.data_ptr(), on.ptr))
        if made:
            on.keep(out)
    return out


def attention_prompt(q, k, v, cu_seqlens, scale=None, out=None, status=None, stream=None):
    """Causal attention of packed prompts: q [n_tokens, n_heads, head_dim], k
    and v [n_tokens, n_kv_heads, head_dim] in float16 or bfloat16, sequence s
    in rows [cu_seqlens[s], cu_seqlens[s+1]); returns q's shape."""
    dev = q.device
    _need(q.is_cuda and q.dim() == 3 and k.dim() == 3, "q, k and v must be 3-D CUDA tensors")
    n, heads, d = q.shape
    _need(q.dtype == k.dtype == v.dtype, "q, k and v must have one type")
    qs, ks = _rows(q, "q", dev, (n, heads, d)), _rows(k, "k", dev, (n, None, d))
    vs = _rows(v, "v", dev, k.shape)
    _ints(cu_seqlens, "cu_seqlens", 1)
    _need(cu_seqlens.device == dev and cu_seqlens.shape[0] >= 1 and cu_seqlens.is_contiguous(), "cu_seqlens must be contiguous, n_seqs + 1 values")
    if status is not None:
        _ints(status, "status", 1)
        _need(status.device == dev, f"status must be on {dev}")
    with _On(dev, stream) as on:
        made = out is None
        out = _result(out, q.shape, q.dtype, dev, "out")
        _check(lib().rpgc_attention_prompt(_type(q), q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs,
                                           cu_seqlens.data_ptr(), cu_seqlens.shape[0] - 1, n, heads, k.shape[1], d,
                                           d ** -0.5 if scale is None else scale, out.data_ptr(),
                                           None if status is None else status.data_ptr(), on.ptr))
        if made:
            on.keep(out)
    return out


def rope_table(positions: int, head_dim: int, theta: float = 1e6, device="cuda"):
    """fp32 [positions, head_dim]: head_dim/2 cosines, then head_dim/2 sines of
    position * theta^(-2i/head_dim), computed in double as BuildRopeTable does
    (src/model.cc:122-145)."""
    import numpy as np
    import torch
    inv = np.array([1.0 / math.pow(theta, 2.0 * i / head_dim) for i in range(head_dim // 2)])
    ang = np.arange(positions, dtype=np.float64)[:, None] * inv
    return torch.from_numpy(np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)).to(device)
