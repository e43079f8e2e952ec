"""The serving operators where calls, memory and odd values meet, on a B200, against 64-bit restatements.

Tolerances are those of test_gpu_serving.py, by the same arithmetic.
"""


import pytest
import torch

from test_gpu_serving import _filled, _gen, _i32
from tiktoktechjam2026track3_b200 import _capi, serving

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _clean_status(cuda_device):
    _capi.device_status(clear=True)
    yield
    torch.cuda.synchronize()
    assert _capi.device_status(clear=True) == 0


def _wide(seqs, page, room=1 << 17):
    """The page table with columns for `room` tokens: heads are then cut into stretches, which need the workspace."""
    return torch.nn.functional.pad(seqs.table, (0, room // page - seqs.table.shape[1]), value=-1).cuda()


# ---------------------------------------------------------------------------------- workspaces
def test_graph_captured_on_its_warm_up_stream_outlives_the_streams_workspace():
    """Warm-up and capture on one stream, then a larger call there, whose workspace takes the place of the smaller one;
    what is allocated after that keeps its values through a replay, and the replay its results."""
    lengths = [5000, 300, 4100, 77]
    cache, seqs = _filled(lengths, 32, 2, 64, E4M3, 4)
    table, n = _wide(seqs, 32), _i32(lengths)
    q = torch.randn(4, 8 * 64, generator=_gen(3)).bfloat16().cuda()
    want = cache.attend(q, table, n)
    out = torch.empty_like(q[:1])
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.attend(q[:1], table[:1], n[:1], out=out)
        with torch.cuda.graph(graph, stream=side):
            cache.attend(q[:1], table[:1], n[:1], out=out)
        assert torch.equal(cache.attend(q, table, n), want)
        others = [torch.full((1 << 20,), 7, dtype=torch.uint8, device="cuda") for _ in range(40)]
        out.zero_()
        graph.replay()
        again = cache.attend(q, table, n)
    torch.cuda.synchronize()
    assert torch.equal(out, want[:1]) and torch.equal(again, want)
    assert all(bool((x == 7).all()) for x in others)
