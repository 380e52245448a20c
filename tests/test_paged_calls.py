"""What the Python layer of the paged-cache operators hands to the library:
strides, workspaces, streams.  Tensors are stand-ins with the attributes of
CUDA tensors and the library's calls are recorded, so no GPU is needed."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import rpgbarengine_b200 as rb  # noqa: E402
from rpgbarengine_b200 import paged  # noqa: E402


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


def table_words(batch):
    """The words of the table that the kernels address: row s at s * table_stride."""
    return [s * batch.c.table_stride + j for s in range(batch.c.n_seqs) for j in range(batch.c.max_pages)]


def test_a_table_of_one_expanded_row_stays_inside_its_storage():
    row = torch.tensor([[4, 7, 2]], dtype=torch.int32)
    table = row.expand(5, -1)
    b = rb.PagedBatch(Dev(table), ints([9] * 5))
    words = table_words(b)
    assert max(words) < row.numel()
    assert row.flatten()[words].tolist() == [4, 7, 2] * 5


@pytest.mark.parametrize("width", [1, 3])
def test_tables_keep_their_own_stride(width):
    wide = torch.arange(60, dtype=torch.int32).view(6, 10)
    table = wide[1:5, 2:2 + width]
    b = rb.PagedBatch(Dev(table), ints([1] * 4))
    assert wide.flatten()[12:][table_words(b)].tolist() == table.flatten().tolist()
    # one row has no stride to speak of
    one = torch.empty_strided((1, width), (0, 1), dtype=torch.int32)
    assert rb.PagedBatch(Dev(one), ints([1])).c.table_stride >= width


def test_tables_whose_rows_overlap_are_refused():
    # (the entry point refuses them too: test_paged_args.py)
    table = torch.arange(20, dtype=torch.int32).as_strided((4, 5), (2, 1))
    with pytest.raises(rb.RpgcError) as e:
        rb.PagedBatch(Dev(table), ints([1] * 4))
    assert e.value.code == rb.E_ARG and "block_table" in str(e.value)


def test_the_entry_point_takes_a_row_that_all_sequences_share():
    # stride 0 passes the batch's checks: the call is refused for the scale alone
    p = 1 << 20
    s3 = (C.c_int64 * 3)(16 * 8 * 128, 8 * 128, 128)
    kv = paged._KV(p, p, s3, s3, rb.F16, 10, 16, 8, 128)
    for stride, word in ((0, "scale"), (4, "scale"), (1, "table_stride"), (-4, "table_stride")):
        b = paged._Batch(p, stride, 4, 2, p, None, 2, None)
        rc = rb.lib().rpgc_paged_attention_decode(C.byref(kv), C.byref(b), p, paged._S2(1024, 128), 16, 0.0, p, p, 1 << 40, None)
        assert rc == rb.E_ARG and word in rb.lib().rpgc_last_error().decode()


# ------------------------------------------------------------ streams
class Recorder:
    """torch and the library as paged.py uses them around a decode call: which stream is
    current when memory is made, which memory and stream each launch gets."""
    uint8, int32 = torch.uint8, torch.int32

    def __init__(self):
        self.current, self.capturing, self.made, self.launches, outer = 0, set(), {}, [], self

        class Stream:
            def __init__(self, handle):
                self.cuda_stream = handle

        class On:
            def __init__(self, stream):
                self.new = stream.cuda_stream

            def __enter__(self):
                self.old, outer.current = outer.current, self.new

            def __exit__(self, *_):
                outer.current = self.old

        class Nothing:
            def __init__(self, *_):
                pass

            __enter__ = __exit__ = lambda *_: None

        class Cuda:
            device, stream = Nothing, On
            ExternalStream = staticmethod(lambda handle, device=None: Stream(handle))
            default_stream = staticmethod(lambda device=None: Stream(0))
            current_stream = staticmethod(lambda device=None: Waits(outer.current))
            is_current_stream_capturing = staticmethod(lambda: outer.current in outer.capturing)

        class Waits(Stream):
            def synchronize(self):
                assert self.cuda_stream not in outer.capturing, "waits inside a capture"

        class Raw:
            _cuda_getDevice = staticmethod(lambda: 0)
            _cuda_getCurrentRawStream = staticmethod(lambda index: outer.current)

        self.cuda, self._C, self.On, self.Stream = Cuda, Raw, On, Stream

    def zeros(self, n, **_):
        t = torch.zeros(n, dtype=torch.uint8)
        self.made[t.data_ptr()] = (self.current, t)
        return t

    def rpgc_paged_decode_workspace(self, kv, n_seqs, n_heads):
        return 64 * n_heads

    def rpgc_paged_attention_decode(self, kv, b, q, st, heads, scale, out, ws, ws_bytes, stream):
        assert ws_bytes == 64 * heads
        self.launches.append((ws, stream))
        return 0


@pytest.fixture
def recorder(monkeypatch):
    r = Recorder()
    monkeypatch.setattr(paged, "_torch", lambda: r)
    monkeypatch.setattr(paged, "lib", lambda: r)
    return r


def decode_inputs():
    class Cache:
        dtype, index, n_kv_heads, head_dim, scale, ref = torch.bfloat16, 0, 2, 64, 0.125, None

    q = Dev(torch.zeros(3, 4, 64, dtype=torch.bfloat16))
    out = Dev(torch.zeros(3, 4, 64, dtype=torch.bfloat16))
    return Cache, rb.PagedBatch(ints([[0, 1]] * 3), ints([5] * 3)), q, out


def test_a_workspace_is_used_on_the_stream_that_owns_its_memory_alone(recorder):
    # memory goes back to the stream that it was made on when the batch is dropped: a call
    # still running on another would share it with whatever the allocator puts there
    cache, batch, q, out = decode_inputs()
    rb.paged_attention_decode(cache, batch, q, out=out)
    rb.paged_attention_decode(cache, batch, q, out=out, stream=0x50)
    with recorder.On(recorder.Stream(0x70)):
        rb.paged_attention_decode(cache, batch, q, out=out)
        rb.paged_attention_decode(cache, batch, q, out=out, stream=0)
    rb.paged_attention_decode(cache, batch, q, out=out)
    assert [s for _, s in recorder.launches] == [0, 0x50, 0x70, 0, 0]
    for ws, stream in recorder.launches:
        assert recorder.made[ws][0] == stream
    assert len(recorder.made) == 3  # (made once per stream)


def test_a_captured_call_uses_a_workspace_that_is_there(recorder):
    cache, batch, q, out = decode_inputs()
    recorder.capturing.add(0x90)
    with recorder.On(recorder.Stream(0x90)):
        with pytest.raises(rb.RpgcError) as e:  # nothing is made or waited for inside a capture
            rb.paged_attention_decode(cache, batch, q, out=out)
    assert e.value.code == rb.E_STATE and not recorder.made and not recorder.launches
    rb.paged_attention_decode(cache, batch, q, out=out)
    with recorder.On(recorder.Stream(0x90)):
        rb.paged_attention_decode(cache, batch, q, out=out)
    assert recorder.launches[1] == (recorder.launches[0][0], 0x90) and len(recorder.made) == 1


@pytest.mark.parametrize("handle", [0, 0x50])
def test_a_result_outlives_its_use_on_the_stream_that_was_asked_for(recorder, monkeypatch, handle):
    # made on the current stream, written on another, the default one (handle 0) among them
    cache, batch, q, out = decode_inputs()
    recorded = []
    out.record_stream, out.device = lambda s: recorded.append(s.cuda_stream), "cuda:0"
    pool = iter(range(0x1000, 0x2000))
    monkeypatch.setattr(recorder.cuda, "ExternalStream",  # (as torch has it: no handle, a stream of the pool)
                        staticmethod(lambda handle, device=None: recorder.Stream(handle or next(pool))))
    monkeypatch.setattr(paged, "_new", lambda like, dtype=None: out)
    with recorder.On(recorder.Stream(0x70)):
        rb.paged_attention_decode(cache, batch, q, stream=handle)
    assert recorder.launches[-1][1] == handle and recorded == [handle]


def test_the_status_of_calls_without_a_word_of_their_own_can_be_asked_for():
    assert rb.lib().rpgc_paged_status(None) == rb.E_ARG
    assert "bits is NULL" in rb.lib().rpgc_last_error().decode()
    assert callable(rb.paged_status)
