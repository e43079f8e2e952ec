"""StreamingTransformer on a B200: what happens around its passes (weights that change, captures, autograd modes)."""

import pytest
import torch

from test_gpu_streaming import _model, _x
from tiktoktechjam2026track3_b200 import StreamingTransformer, rotary_table

pytestmark = pytest.mark.gpu


def _talk(stream, seed=1):
    """A prompt of two ragged sequences, then three steps."""
    d = stream.config.d_model
    outs = [stream.prompt(_x(2, 40, d, seed).cuda(), [40, 11])]
    outs += [stream.step(_x(2, t, d, seed + t).cuda()) for t in (1, 2, 1)]
    return outs


def _make(model, graphs):
    stream = StreamingTransformer(model, 2, 64, table=rotary_table(64, 64), window=30, sinks=2)
    stream.use_cuda_graph = graphs
    return stream


def _scaled(t):
    return t * 1.25 + 0.01


def _in_place(model):
    for p in model.parameters():
        p.copy_(_scaled(p))


def _final_norm_only(model):
    model.final_norm.weight.copy_(_scaled(model.final_norm.weight))


def _new_storage(model):
    for p in model.parameters():
        p.data = _scaled(p.data)


def _new_parameters(model):
    for layer in model.layers:
        layer.ffn_in.weight = torch.nn.Parameter(_scaled(layer.ffn_in.weight.detach()))


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("change", [_in_place, _final_norm_only, _new_storage, _new_parameters])
@torch.no_grad()
def test_passes_use_the_weights_as_they_are(cuda_device, graphs, change):
    """After a change the next conversation is a fresh object's; memory of the old weights is filled with NaN first."""
    model, _ = _model(256, 4)
    stream = _make(model, graphs)
    before = _talk(stream)
    change(model)
    junk = [torch.full((1 << 18,), float("nan"), device="cuda") for _ in range(16)]  # takes freed storage, if there is any
    got, want = _talk(stream), _talk(_make(model, graphs))
    for a, b, c in zip(got, want, before):
        assert torch.equal(a, b) and not torch.equal(a, c)
    del junk


@torch.no_grad()
def test_a_step_sees_weights_changed_in_the_middle_of_a_conversation(cuda_device):
    """With graphs as without: the keys and values in the cache stay, all else is the new weights'."""
    got = []
    for graphs in (True, False):
        model, _ = _model(256, 4)
        stream = _make(model, graphs)
        outs = _talk(stream)
        _in_place(model)
        outs += [stream.step(_x(2, 1, 256, 20 + i).cuda()) for i in range(3)]
        got.append(outs)
    for a, b in zip(*got):
        assert torch.equal(a, b)


@torch.no_grad()
def test_passes_refuse_to_be_captured(cuda_device):
    """A first pass would leave buffers that only the graph's replay fills; the conversation goes on as if not asked."""
    model, _ = _model(256, 4)
    want = _talk(_make(model, True))
    for graphs in (True, False):
        stream = _make(model, graphs)
        x = _x(2, 40, 256, 1).cuda()
        for call in (lambda: stream.prompt(x, [40, 11]), lambda: stream.step(x[:, :1])):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                with pytest.raises(RuntimeError, match="captured"):
                    call()
                x.add(1)  # a graph of something
            assert stream.lengths == [0, 0] and not stream._starts and not stream._workspaces
        for a, b in zip(_talk(stream), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("graphs", [True, False])
def test_any_autograd_mode_may_make_and_use_it(cuda_device, graphs):
    """Made or first used under inference mode and then without it, and the other way round; inputs that need gradients
    (the passes have none: their outputs do not, and nothing of a conversation is kept for them)."""
    model, _ = _model(256, 4)
    want = _talk(_make(model, graphs))
    for make, first, then in ((True, True, False), (False, True, False), (True, False, True), (False, False, True)):
        with torch.inference_mode(make):
            stream = _make(model, graphs)
        for mode in (first, then):
            with torch.inference_mode(mode):
                for a, b in zip(_talk(stream), want):
                    assert torch.equal(a, b)
    x = _x(2, 40, 256, 1).cuda().requires_grad_()
    y = stream.prompt(x, [40, 11])
    z = stream.step(x[:, :1] * 1.0)
    assert torch.equal(y, want[0]) and not y.requires_grad and not z.requires_grad
    assert not any(t.requires_grad for g in stream._graphs.values() for t in g[:2])
