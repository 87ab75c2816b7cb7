"""The dense attention block's buffers on streams of the caller's."""
import pytest
import torch

from tests.dense_block import pages, state
from wsvd_b200 import ops

pytestmark = pytest.mark.gpu

F16 = torch.float16


def _calls(stream):
    """Each operator on `stream`, with an output of its own of several megabytes: (output's bytes, call)."""
    g = torch.Generator().manual_seed(1)
    table, T = pages(2, 4000, 16, g)
    st = state([0, 0], table, device="cuda")
    cache = [torch.zeros(T, 2, 128, dtype=F16, device="cuda") for _ in range(2)]
    kv, q = torch.zeros(3000, 2, 128, dtype=F16, device="cuda"), torch.zeros(3000, 8, 128, dtype=F16, device="cuda")
    cu = torch.tensor([0, 2000, 3000], dtype=torch.int32, device="cuda")
    yield q.nbytes, lambda: ops.kv_rope_append(kv, kv, st, *cache, torch.zeros(64, device="cuda"), q=q, cu_new=cu, stream=stream)
    many = state([3] * 2000, table[:1].expand(2000, -1).contiguous(), device="cuda")
    yield q[:2000].nbytes, lambda: ops.paged_decode(q[:2000], many, *cache, stream=stream)
    y = torch.zeros(3000, 1024, dtype=F16, device="cuda")
    a, b = torch.zeros(1, 64, 8, dtype=F16, device="cuda"), torch.zeros(1, 8, 1024, dtype=F16, device="cuda")
    none = torch.zeros(2, dtype=torch.int32, device="cuda")
    yield y.nbytes, lambda: ops.adapter_add(y, y[:, :64], a, b, none, cu_new=cu, stream=stream)


def test_buffers_for_another_stream_are_not_the_current_streams():
    """What has just gone back to the current stream's pool may still be read there: it is not what a call on another stream writes to."""
    side = torch.cuda.Stream()
    for size, call in _calls(side):
        side.wait_stream(torch.cuda.current_stream())
        torch.cuda.synchronize()
        freed = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(3)]
        used = [(t.data_ptr(), t.data_ptr() + t.nbytes) for t in freed]
        del freed
        out = call()
        assert not any(first <= out.data_ptr() < last for first, last in used)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()


def test_an_output_from_another_stream_is_not_handed_out_while_the_current_one_reads_it():
    side = torch.cuda.Stream()
    for size, call in _calls(side):
        side.wait_stream(torch.cuda.current_stream())
        out = call()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda._sleep(200_000_000)  # (some 100 ms: the current stream has not come to the end of its work)
        reader = out.clone()
        where = out.data_ptr()
        del out
        with torch.cuda.stream(side):
            again = torch.empty(size, dtype=torch.uint8, device="cuda")
        assert again.data_ptr() != where
        torch.cuda.synchronize()
        del reader, again
