"""StreamingTransformer on a B200: prompts and steps against a 64-bit stack on the same bf16 weights and inputs.

The gate is the model's own, max|y - r| <= 2^-7 max|r|; over an 8-bit cache each key and value is off by up to 2^-4 of itself,
and the output may move by that share.
"""

import pytest
import torch

from oracle import reference_fp32, serving_fp64
from tiktoktechjam2026track3_b200 import StreamingTransformer, TransformerConfig, UserOptimizedTransformer, rotary_table

pytestmark = pytest.mark.gpu


def _model(d_model, heads, layers=2):
    cfg = TransformerConfig(3, 64, d_model, heads, 4 * d_model, layers, True)
    state = reference_fp32.round_state_to_bf16(reference_fp32.build_reference_state(cfg, 0))
    model = UserOptimizedTransformer(cfg)
    model.load_state_dict(state, strict=True)
    return model.to(device="cuda", dtype=torch.bfloat16).eval(), state


def _x(batch, tokens, d, seed):
    return torch.randn(batch, tokens, d, generator=torch.Generator().manual_seed(seed)).bfloat16()


def _gate(got, ref, limit):
    got, ref = got.double().cpu(), ref.double()
    assert bool(torch.isfinite(got).all())
    assert float((got - ref).abs().max()) <= limit * float(ref.abs().max())


CASES = [
    # d_model, heads, rotary_dim, interleaved, window, sinks, dtype, page_size
    (256, 4, 0, False, 0, 0, torch.bfloat16, 16),
    (256, 4, 64, False, 0, 0, torch.float8_e4m3fn, 64),
    (256, 2, 128, True, 24, 4, torch.bfloat16, 32),
    (256, 2, 64, False, 24, 4, torch.float8_e4m3fn, 16),
    (128, 4, 32, True, 40, 0, torch.bfloat16, 64),
]


@pytest.mark.parametrize("d,heads,rotary_dim,interleaved,window,sinks,dtype,page", CASES)
@torch.inference_mode()
def test_prompt_and_steps(cuda_device, d, heads, rotary_dim, interleaved, window, sinks, dtype, page):
    model, state = _model(d, heads)
    table = rotary_table(256, rotary_dim) if rotary_dim else None
    stream = StreamingTransformer(model, 3, 200, table=table, interleaved=interleaved, window=window, sinks=sinks,
                                  page_size=page, dtype=dtype)
    lengths, steps = [70, 1, 33], [1, 1, 3, 1]
    prompt, more = _x(3, 70, d, 1), _x(3, sum(steps), d, 2)
    outs = [stream.prompt(prompt.cuda(), lengths)]
    at = 0
    for t in steps:
        outs.append(stream.step(more[:, at:at + t].cuda()))
        at += t
    stream.check_device_status()
    after = torch.cat(outs[1:], 1)
    for b, n in enumerate(lengths):
        whole = torch.cat([prompt[b, :n], more[b]]).double()
        ref = serving_fp64.stack(state, heads, 2, whole, table.cpu() if rotary_dim else None, rotary_dim, interleaved, window,
                                 sinks)
        _gate(outs[0][b, :n], ref[:n], 2**-7)
        assert not bool(outs[0][b, n:].any())
        _gate(after[b], ref[n:], 2**-7 if dtype == torch.bfloat16 else 2**-4)


@torch.inference_mode()
def test_graphs_and_eager_launches_agree(cuda_device):
    model, _ = _model(256, 4)
    table = rotary_table(128, 64)
    got = []
    for graphs in (True, False):
        stream = StreamingTransformer(model, 2, 128, table=table, window=30, sinks=2)
        stream.use_cuda_graph = graphs
        outs = [stream.prompt(_x(2, 50, 256, 1).cuda(), [50, 20])]
        outs += [stream.step(_x(2, 1, 256, 10 + i).cuda()) for i in range(20)]
        stream.reset()  # a second conversation on the same caches
        outs += [stream.prompt(_x(2, 9, 256, 3).cuda()), stream.step(_x(2, 2, 256, 4).cuda())]
        got.append(outs)
    for a, b in zip(*got):
        assert torch.equal(a, b)


@torch.inference_mode()
def test_prompt_is_the_models_forward(cuda_device):
    """Without positions and a window the prompt pass computes what the model's causal forward does."""
    model, _ = _model(256, 2)
    x = _x(3, 150, 256, 5).cuda()
    stream = StreamingTransformer(model, 3, 150, dtype=torch.bfloat16)
    y, ref = stream.prompt(x), model(x)
    assert float((y.float() - ref.float()).abs().max()) <= 2**-7 * float(ref.float().abs().max())


@torch.inference_mode()
def test_refusals(cuda_device):
    model, _ = _model(256, 4)
    stream = StreamingTransformer(model, 2, 20)
    with pytest.raises(ValueError, match="fit"):
        stream.prompt(_x(2, 21, 256, 0).cuda())
    with pytest.raises(ValueError, match="lengths"):
        stream.prompt(_x(2, 5, 256, 0).cuda(), [6, 1])
    with pytest.raises(ValueError, match="x must be"):
        stream.step(_x(3, 1, 256, 0).cuda())
    with pytest.raises(RuntimeError, match="GPU"):
        stream.step(_x(2, 1, 256, 0))
    stream.prompt(_x(2, 20, 256, 0).cuda())
    with pytest.raises(ValueError, match="fit"):
        stream.step(_x(2, 1, 256, 0).cuda())
