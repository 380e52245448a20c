"""Paged-cache operators at the edges of their contract.

Where two calls do the same arithmetic on the same visible values their results
are compared bit for bit; else against 64 bits with the bounds of
test_gpu_paged.py."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import rpgbarengine_b200 as rb  # noqa: E402
from test_gpu_paged import check_decode, decode_case, i32  # noqa: E402


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
