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
