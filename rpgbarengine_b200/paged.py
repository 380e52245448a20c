"""Paged KV cache on the device (rpgc_paged_*, rpgc_paged8_*, rpgc_attention_prompt).

  PagedKV                  one layer's K and V pools: [page, position, kv head, head_dim]
  PagedKV8                 the same in 8 bits: e4m3 codes and a scale for each row
  PagedBatch               the sequences of a call: block table, lengths, packed rows
  PagedPrefix              first positions that groups of sequences share
  paged_append             QK-norm + RoPE + write of new tokens into their pages
  paged_attention_decode   one new token per sequence over its pages
  paged_read               positions of 8-bit pages back into 16-bit pages
  paged_attention_prompt   causal attention of packed prompts over their pages
  attention_prompt         the same with K and V packed beside q
  rope_table               the cosine and sine rows paged_append reads
  paged_status             what calls without a status word have reported

Lengths, tables and page ids live on the device and are read there when the
call runs: nothing here but paged_status waits for the GPU, and all calls can
be captured (decode's once its batch has a workspace, which an earlier call makes).
"""
from __future__ import annotations

import ctypes as C
import math

from . import BF16, E_ARG, E_STATE, F16, F32, RpgcError, _check, lib

DROPPED, TIMEOUT = 1, 2  # PagedBatch.status bits


class _KV(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_stride", C.c_int64 * 3), ("v_stride", C.c_int64 * 3),
                ("type", C.c_uint32), ("n_pages", C.c_int32), ("page_size", C.c_int32),
                ("n_kv_heads", C.c_int32), ("head_dim", C.c_int32)]


class _Batch(C.Structure):
    _fields_ = [("block_table", C.c_void_p), ("table_stride", C.c_int64), ("max_pages", C.c_int32),
                ("n_seqs", C.c_int32), ("kv_lens", C.c_void_p), ("cu_q", C.c_void_p),
                ("n_tokens", C.c_int64), ("status", C.c_void_p)]


class _KV8(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_stride", C.c_int64 * 3), ("v_stride", C.c_int64 * 3),
                ("scales", C.c_void_p), ("scale_stride", C.c_int64 * 2), ("type", C.c_uint32), ("n_pages", C.c_int32),
                ("page_size", C.c_int32), ("n_kv_heads", C.c_int32), ("head_dim", C.c_int32)]


class _Prefix(C.Structure):
    _fields_ = [("kv", C.POINTER(_KV)), ("block_table", C.c_void_p), ("table_stride", C.c_int64), ("max_pages", C.c_int32),
                ("n_groups", C.c_int32), ("lens", C.c_void_p), ("cu_seqs", C.c_void_p)]


_S2 = C.c_int64 * 2
_strides = {}  # (token, head) strides -> their C array
_mods = []


def _torch():
    if not _mods:
        import torch
        _mods.append(torch)
    return _mods[0]


def _refuse(msg):
    raise RpgcError(E_ARG, msg)


def _need(ok, msg):
    if not ok:
        _refuse(msg)


def _type(t):
    torch = _torch()
    d = t.dtype
    return BF16 if d is torch.bfloat16 else F16 if d is torch.float16 else F32 if d is torch.float32 else \
        _refuse(f"{d} is not supported")


def _ints(t, what, dims):
    _need(t.is_cuda and t.dtype is _torch().int32 and t.dim() == dims, f"{what} must be a {dims}-D int32 CUDA tensor")


def _rows(t, what, index, n, heads, d):
    """Strides of a [token, head, dim] tensor with contiguous rows on device `index`."""
    shape, st = t.shape, t.stride()
    if t.get_device() != index or len(shape) != 3 or shape[0] != n or shape[2] != d or (heads and shape[1] != heads) or st[2] != 1:
        _refuse(f"{what} must be [{n}, {heads or 'heads'}, {d}] on CUDA device {index}, each row of {d} contiguous; "
                f"got {tuple(shape)} with strides {tuple(st)} on {t.device}")
    # (a dimension of one has no stride to speak of)
    key = st[0] if n > 1 else shape[1] * d, st[1] if shape[1] > 1 else d
    c = _strides.get(key)
    if c is None:
        if len(_strides) > 1000:
            _strides.clear()
        c = _strides[key] = _S2(*key)
    return c


def _table(t, what, n):
    """Row stride and width of a block table of n rows."""
    _ints(t, what, 2)
    width = t.shape[1]
    stride = t.stride(0) if n > 1 else width  # (one row has no stride to speak of)
    _need(t.shape[0] == n and (t.stride(1) == 1 or width < 2), f"{what} needs one contiguous row per sequence")
    _need(stride == 0 or stride >= width, f"{what}'s rows overlap: they must be apart, or one row expanded to all sequences")
    return stride, width


def _new(like, dtype=None):
    """A contiguous tensor of `like`'s shape (the cheapest call that makes one)."""
    torch = _torch()
    if dtype is None and like.is_contiguous():
        return torch.empty_like(like)
    return torch.empty_like(like, dtype=dtype, memory_format=torch.contiguous_format)


def _result(out, like, shape, dtype):
    if out.shape != shape or out.dtype != dtype or out.get_device() != like.get_device() or not out.is_contiguous():
        _refuse(f"out must be a contiguous {dtype} tensor of shape {tuple(shape)} on {like.device}")
    return out


def _on(index, stream):
    """The stream of a call on device `index`, or None where another device is current."""
    c = _torch()._C
    if c._cuda_getDevice() != index:
        return None
    return c._cuda_getCurrentRawStream(index) if stream is None else int(stream)


def _stream_at(index, handle):
    """The stream of a handle (torch makes a new one of handle 0, which is the default stream)."""
    cuda = _torch().cuda
    return cuda.ExternalStream(handle, device=index) if handle else cuda.default_stream(index)


def _run(fn, index, stream, made, *args):
    """fn(*args, stream) with device `index` current.  `made`: a result allocated
    here, whose memory must outlive its use on a stream that is not the current one."""
    ptr = _on(index, stream)
    if ptr is None:
        with _torch().cuda.device(index):
            return _run(fn, index, stream, made, *args)
    rc = fn(*args, ptr)
    if rc < 0:
        _check(rc)
    if made is not None and stream is not None:
        made.record_stream(_stream_at(index, ptr))


class PagedKV:
    """One layer's K and V pools, [n_pages, page_size, n_kv_heads, head_dim]
    in float16 or bfloat16, any strides that are multiples of 8 elements (a
    head-major pool is passed transposed).  Holds references to both."""

    def __init__(self, k, v):
        _need(k.is_cuda and k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype and k.device == v.device,
              "k and v must be 4-D CUDA tensors of one shape and type")
        _need(k.stride(3) == 1 and v.stride(3) == 1, "rows of head_dim values must be contiguous")
        self.k, self.v, self.index, self.dtype = k, v, k.get_device(), k.dtype
        n, p, h, d = k.shape
        ty = _type(k)
        _need(ty != F32, "a paged cache holds float16 or bfloat16")
        strides = [(C.c_int64 * 3)(*[st if size > 1 else d for st, size in zip(t.stride(), t.shape[:3])]) for t in (k, v)]
        self.c = _KV(k.data_ptr(), v.data_ptr(), strides[0], strides[1], ty, n, p, h, d)
        self.ref = C.byref(self.c)
        self.page_size, self.n_kv_heads, self.head_dim, self.scale = p, h, d, d ** -0.5

    @classmethod
    def empty(cls, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, dtype=None, device="cuda") -> "PagedKV":
        """New pools (bfloat16 unless said otherwise); their values are never
        read before append writes them."""
        torch = _torch()
        shape, dt = (n_pages, page_size, n_kv_heads, head_dim), dtype or torch.bfloat16
        return cls(torch.empty(shape, dtype=dt, device=device), torch.empty(shape, dtype=dt, device=device))


class PagedKV8:
    """One layer's K and V pools in 8 bits: k and v float8_e4m3fn [n_pages,
    page_size, n_kv_heads, head_dim] codes, any strides that are multiples of 16,
    and scales float32 [n_pages, n_kv_heads, 2, page_size] (K's, then V's; a
    page and head's contiguous): a row's values are scale * code.  dtype: the
    type of q and of attention's results (float16 or bfloat16).  Holds
    references to all three."""

    def __init__(self, k, v, scales, dtype=None):
        torch = _torch()
        _need(k.is_cuda and k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype == torch.float8_e4m3fn and k.device == v.device,
              "k and v must be 4-D CUDA tensors of one shape, float8_e4m3fn")
        _need(k.stride(3) == 1 and v.stride(3) == 1, "rows of head_dim codes must be contiguous")
        n, p, h, d = k.shape
        _need(scales.device == k.device and scales.dtype is torch.float32 and scales.shape == (n, h, 2, p) and
              scales.stride(3) == 1 and scales.stride(2) == p,
              f"scales must be float32 [{n}, {h}, 2, {p}] on the pools' device, the last two dimensions contiguous")
        self.k, self.v, self.scales, self.index = k, v, scales, k.get_device()
        self.dtype = dtype or torch.bfloat16
        _need(self.dtype in (torch.float16, torch.bfloat16), "dtype must be float16 or bfloat16")
        strides = [(C.c_int64 * 3)(*[st if size > 1 else d for st, size in zip(t.stride(), t.shape[:3])]) for t in (k, v)]
        st = _S2(scales.stride(0) if n > 1 else 2 * h * p, scales.stride(1) if h > 1 else 2 * p)
        self.c = _KV8(k.data_ptr(), v.data_ptr(), strides[0], strides[1], scales.data_ptr(), st,
                      BF16 if self.dtype is torch.bfloat16 else F16, n, p, h, d)
        self.ref = C.byref(self.c)
        self.page_size, self.n_kv_heads, self.head_dim, self.scale = p, h, d, d ** -0.5

    @classmethod
    def empty(cls, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, dtype=None, device="cuda") -> "PagedKV8":
        """New pools; their values are never read before append writes them."""
        torch = _torch()
        shape = (n_pages, page_size, n_kv_heads, head_dim)
        return cls(torch.empty(shape, dtype=torch.float8_e4m3fn, device=device), torch.empty(shape, dtype=torch.float8_e4m3fn, device=device),
                   torch.empty((n_pages, n_kv_heads, 2, page_size), dtype=torch.float32, device=device), dtype)


class PagedPrefix:
    """First positions that groups of a batch's sequences share, for
    paged_attention_decode.  Group g is sequences [cu_seqs[g], cu_seqs[g+1]) of the
    batch (those outside all groups share nothing); its sequences' positions
    [0, lens[g]) are read once for all of them, through row g of block_table
    (int32 [n_groups, max_pages]) from `cache`, a PagedKV: the batch's own, where
    the sequences name the same pages, or another (for a batch in 8 bits, one that
    paged_read has filled).  The sequences' own tables' entries for those
    positions are not looked at.  lens [n_groups], cu_seqs [n_groups + 1]:
    int32, on the device like the table, and read there at each call.  Holds
    references to all of them."""

    def __init__(self, cache: PagedKV, block_table, lens, cu_seqs):
        _need(isinstance(cache, PagedKV), "a prefix lies in a PagedKV (16 bits)")
        _ints(lens, "lens", 1)
        _ints(cu_seqs, "cu_seqs", 1)
        n = lens.shape[0]
        stride, width = _table(block_table, "block_table", n)
        _need(lens.stride(0) == 1 or n < 2, "lens must be contiguous")
        _need(cu_seqs.shape[0] == n + 1 and cu_seqs.is_contiguous(), "cu_seqs must hold n_groups + 1 contiguous values")
        self.index, self.cache, self.keep = cache.index, cache, (block_table, lens, cu_seqs)
        _need(all(t.get_device() == self.index for t in self.keep), "the prefix's tensors must be on its cache's device")
        self.c = _Prefix(C.pointer(cache.c), block_table.data_ptr(), stride, width, n, lens.data_ptr(), cu_seqs.data_ptr())
        self.ref = C.byref(self.c)


class PagedBatch:
    """The sequences of a call.  block_table: int32 [n_seqs, max_pages] page
    ids (one row expanded to n_seqs: all sequences over the same pages);
    kv_lens: int32 [n_seqs] cache lengths, the call's new tokens included;
    cu_q: int32 [n_seqs + 1], sequence s's new tokens are rows
    [cu_q[s], cu_q[s+1]) of n_tokens (None: one new token per sequence).  All on
    the device, and read there at each call, so a decode loop updates them in
    place and keeps the batch.  status: int32 tensor of one word that
    receives DROPPED / TIMEOUT bits (None: see paged_status).

    The batch also holds decode's workspaces, one for each stream that it is
    used on, made by the first call there.  A captured call uses one that is
    there already (of a call outside the graph), so the batch is kept until the
    graph's last replay has ended, and replays are ordered with each other and with
    other calls on that stream."""

    def __init__(self, block_table, kv_lens, cu_q=None, n_tokens=None, status=None):
        _ints(kv_lens, "kv_lens", 1)
        n = kv_lens.shape[0]
        stride, width = _table(block_table, "block_table", n)
        _need(kv_lens.stride(0) == 1 or n < 2, "kv_lens must be contiguous")
        if cu_q is not None:
            _ints(cu_q, "cu_q", 1)
            _need(cu_q.shape[0] == n + 1 and cu_q.stride(0) == 1, "cu_q must hold n_seqs + 1 contiguous values")
            _need(n_tokens is not None, "n_tokens is needed with cu_q")
        if status is not None:
            _ints(status, "status", 1)
        self.keep = (block_table, kv_lens, cu_q, status)
        self.index = kv_lens.get_device()
        _need(all(t is None or t.get_device() == self.index for t in self.keep), "the batch's tensors must be on one device")
        self.n_seqs, self.n_tokens = n, n if n_tokens is None else int(n_tokens)
        p = [None if t is None else t.data_ptr() for t in self.keep]
        self.c = _Batch(p[0], stride, width, n, p[1], p[2], self.n_tokens, p[3])
        self.ref = C.byref(self.c)
        self._ws = {}

    def workspace(self, cache, n_heads: int, stream: int, prefix: bool = False):
        """Decode's workspace for this batch, head count and stream, with a
        prefix or without (made once).  It is zeroed and used on that stream, and its memory is the
        stream's: when the batch is dropped, what gets it next runs after the
        calls that are still using it."""
        shape = (n_heads, cache.n_kv_heads, cache.head_dim) + (("prefix",) if prefix else ())
        ws = self._ws.get((shape, stream))
        if ws is None:
            torch = _torch()
            with torch.cuda.device(self.index), torch.cuda.stream(_stream_at(self.index, stream)):
                if torch.cuda.is_current_stream_capturing():
                    for key, ws in self._ws.items():
                        if key[0] == shape:
                            return ws
                    raise RpgcError(E_STATE, "a captured decode call needs the workspace of an earlier one on its batch: make a call outside the graph first")
                n = _check(lib().rpgc_paged_prefix_workspace(self.n_seqs, n_heads, cache.n_kv_heads, cache.head_dim) if prefix else
                           lib().rpgc_paged8_decode_workspace(cache.ref, self.n_seqs, n_heads) if isinstance(cache, PagedKV8) else
                           lib().rpgc_paged_decode_workspace(cache.ref, self.n_seqs, n_heads))
                buf = torch.zeros(n, dtype=torch.uint8, device="cuda")
            ws = self._ws[shape, stream] = (buf, buf.data_ptr(), n)
        return ws


def paged_append(cache, batch: PagedBatch, q, k, v, q_norm=None, k_norm=None, eps: float = 1e-6, rope=None,
                 q_out=None, stream=None):
    """Writes the batch's new tokens into their pages and returns q normalised
    and rotated in the cache's type (None when q is None).  q [n_tokens,
    n_heads, head_dim], k and v [n_tokens, n_kv_heads, head_dim], of one type
    (float32, float16 or bfloat16); q_norm / k_norm: fp32 gains [head_dim] or
    None; rope: fp32 [positions, head_dim] (rope_table) or None.  Rows that no
    sequence holds are zeros in the result and write nothing to the cache.
    cache: a PagedKV or a PagedKV8."""
    torch = _torch()
    index, n, d, kv = cache.index, batch.n_tokens, cache.head_dim, cache.n_kv_heads
    _need(batch.index == index, "cache and batch are on different devices")
    ty = _type(k)
    _need(v.dtype is k.dtype and (q is None or q.dtype is k.dtype), "q, k and v must have one type")
    ks, vs = _rows(k, "k", index, n, kv, d), _rows(v, "v", index, n, kv, d)
    for g in (q_norm, k_norm):
        if g is not None and not (g.get_device() == index and g.dtype is torch.float32 and g.shape == (d,) and g.is_contiguous()):
            _refuse("norm gains must be contiguous float32 [head_dim] on the cache's device")
    if rope is not None and not (rope.get_device() == index and rope.dtype is torch.float32 and rope.dim() == 2 and
                                 rope.shape[1] == d and rope.is_contiguous()):
        _refuse("rope must be contiguous float32 [positions, head_dim] on the cache's device")
    qs, heads, qp, op, made = None, 0, None, None, None
    if q is not None:
        qs, heads, qp = _rows(q, "q", index, n, 0, d), q.shape[1], q.data_ptr()
        if q_out is None:
            q_out = made = _new(q, cache.dtype)
        else:
            _result(q_out, q, q.shape, cache.dtype)
        op = q_out.data_ptr()
    else:
        _need(q_out is None, "q_out without q")
    _run(lib().rpgc_paged8_append if isinstance(cache, PagedKV8) else lib().rpgc_paged_append, index, stream, made, cache.ref, batch.ref, ty, qp, qs, heads, k.data_ptr(), ks, v.data_ptr(), vs,
         None if q_norm is None else q_norm.data_ptr(), None if k_norm is None else k_norm.data_ptr(), eps,
         None if rope is None else rope.data_ptr(), 0 if rope is None else rope.shape[0], op)
    return q_out


def _attend(cache, batch, q, out):
    """Strides of q, the result and whether it was made here."""
    if q.dtype is not cache.dtype or batch.index != cache.index:
        _refuse("q, cache and batch must share their device, and q the cache's type")
    qs = _rows(q, "q", cache.index, batch.n_tokens, 0, cache.head_dim)
    if out is None:
        out = _new(q)
        return qs, out, out
    return qs, _result(out, q, q.shape, q.dtype), None


def paged_attention_decode(cache, batch: PagedBatch, q, scale=None, out=None, stream=None, prefix: PagedPrefix = None):
    """Attention of one new token per sequence, q [n_seqs, n_heads, head_dim],
    over the sequence's positions; returns the same shape.  scale: default
    head_dim ** -0.5.  cache: a PagedKV or a PagedKV8.  prefix: first positions that
    groups of the sequences share, read once for each group; the results are
    those without it, up to rounding, where the sequences name the same pages."""
    qs, out, made = _attend(cache, batch, q, out)
    heads, eight = q.shape[1], isinstance(cache, PagedKV8)
    ws = batch.workspace(cache, heads, _torch()._C._cuda_getCurrentRawStream(cache.index) if stream is None else int(stream),
                         *(() if prefix is None else (True,)))
    scale = cache.scale if scale is None else scale
    if prefix is None and not eight:
        _run(lib().rpgc_paged_attention_decode, cache.index, stream, made, cache.ref, batch.ref, q.data_ptr(), qs, heads, scale,
             out.data_ptr(), ws[1], ws[2])
        return out
    if prefix is not None and prefix.index != cache.index:
        _refuse("cache and prefix are on different devices")
    _run(lib().rpgc_paged8_attention_decode if eight else lib().rpgc_paged_attention_decode_prefix, cache.index, stream, made, cache.ref,
         batch.ref, None if prefix is None else prefix.ref, q.data_ptr(), qs, heads, scale, out.data_ptr(), ws[1], ws[2])
    return out


def paged_read(cache: PagedKV8, batch: PagedBatch, to: PagedKV, to_table, stream=None):
    """Positions [0, kv_lens[s]) of every sequence of the batch, rounded once
    to `to`'s type, into the slots that row s of to_table (int32 [n_seqs,
    pages]) names there: what prompt attention and a PagedPrefix read.
    Positions whose page is not in the batch's table are left out; those without one
    in to_table are dropped (DROPPED in the batch's status)."""
    _need(isinstance(cache, PagedKV8) and isinstance(to, PagedKV), "paged_read goes from a PagedKV8 to a PagedKV")
    stride, width = _table(to_table, "to_table", batch.n_seqs)
    if not cache.index == batch.index == to.index == to_table.get_device():
        _refuse("cache, batch, to and to_table must be on one device")
    _run(lib().rpgc_paged8_read, cache.index, stream, None, cache.ref, batch.ref, to.ref, to_table.data_ptr(), stride, width)


def paged_attention_prompt(cache: PagedKV, batch: PagedBatch, q, scale=None, out=None, stream=None):
    """Causal attention of the batch's new tokens, q [n_tokens, n_heads,
    head_dim], over their sequences' pages (a cached prefix included).  Rows
    that no sequence holds are not written: in a result made here they hold
    anything.  (An 8-bit cache is read back first: paged_read.)"""
    _need(isinstance(cache, PagedKV), "prompt attention reads 16-bit pages: paged_read brings an 8-bit cache's back into some")
    qs, out, made = _attend(cache, batch, q, out)
    _run(lib().rpgc_paged_attention_prompt, cache.index, stream, made, cache.ref, batch.ref, q.data_ptr(), qs, q.shape[1],
         cache.scale if scale is None else scale, out.data_ptr())
    return out


def attention_prompt(q, k, v, cu_seqlens, scale=None, out=None, status=None, stream=None):
    """Causal attention of packed prompts: q [n_tokens, n_heads, head_dim], k
    and v [n_tokens, n_kv_heads, head_dim] in float16 or bfloat16, sequence s
    in rows [cu_seqlens[s], cu_seqlens[s+1]); returns q's shape.  Rows of no
    sequence as in paged_attention_prompt."""
    if not q.is_cuda or q.dim() != 3 or k.dim() != 3 or q.dtype is not k.dtype or q.dtype is not v.dtype:
        _refuse("q, k and v must be 3-D CUDA tensors of one type")
    index, (n, heads, d), kv = q.get_device(), q.shape, k.shape[1]
    qs, ks, vs = _rows(q, "q", index, n, heads, d), _rows(k, "k", index, n, kv, d), _rows(v, "v", index, n, kv, d)
    _ints(cu_seqlens, "cu_seqlens", 1)
    if cu_seqlens.get_device() != index or cu_seqlens.shape[0] < 1 or not cu_seqlens.is_contiguous():
        _refuse("cu_seqlens must be n_seqs + 1 contiguous values on q's device")
    if status is not None:
        _ints(status, "status", 1)
        _need(status.get_device() == index, "status must be on q's device")
    made = None
    if out is None:
        out = made = _new(q)
    else:
        _result(out, q, q.shape, q.dtype)
    _run(lib().rpgc_attention_prompt, index, stream, made, _type(q), q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs,
         cu_seqlens.data_ptr(), cu_seqlens.shape[0] - 1, n, heads, kv, d, d ** -0.5 if scale is None else scale, out.data_ptr(),
         None if status is None else status.data_ptr())
    return out


def paged_status(device=None) -> int:
    """Waits for the device and returns the DROPPED / TIMEOUT bits that calls
    without a status tensor have reported on it since the last time: after
    TIMEOUT the output of one of them is not valid."""
    torch = _torch()
    bits = C.c_int32()
    with torch.cuda.device(device):
        torch.cuda.synchronize()
        _check(lib().rpgc_paged_status(C.byref(bits)))
    return bits.value


def rope_table(positions: int, head_dim: int, theta: float = 1e6, device="cuda"):
    """fp32 [positions, head_dim]: head_dim/2 cosines, then head_dim/2 sines of
    position * theta^(-2i/head_dim), computed in double as BuildRopeTable does
    (src/model.cc:122-145)."""
    import numpy as np
    torch = _torch()
    inv = np.array([1.0 / math.pow(theta, 2.0 * i / head_dim) for i in range(head_dim // 2)])
    ang = np.arange(positions, dtype=np.float64)[:, None] * inv
    return torch.from_numpy(np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)).to(device)
