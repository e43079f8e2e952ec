"""Chunks of conversations through a cache on a B200: append, read and packed_attention one after the other, and
StreamingTransformer.extend, against 64-bit restatements.

The model's gate is its own, max|y - r| <= 2^-7 max|r|, over a bf16 cache. Over 8 bits each key and value is off by up to 2^-4 of
itself; over 4 bits by up to 0.55 steps, a step being at most 2/15 of the largest value of a group, so by up to 0.0734 of that: the
output may move by that share of the largest value in each of the two products of a layer (2^-3 with the gate).
"""

import pytest
import torch

from oracle import reference_fp32, serving_fp64
from tiktoktechjam2026track3_b200 import (StreamingTransformer, TransformerConfig, UserOptimizedTransformer, _capi, rotary_table,
                                          serving)

pytestmark = pytest.mark.gpu

BF16, E4M3, INT4 = torch.bfloat16, torch.float8_e4m3fn, torch.uint8


@pytest.fixture(autouse=True)
def _clean_status(cuda_device):
    _capi.device_status(clear=True)
    yield
    torch.cuda.synchronize()
    assert _capi.device_status(clear=True) == 0


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _starts(lengths):
    return [sum(lengths[:b]) for b in range(len(lengths) + 1)]


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).bfloat16()


def _gate(got, ref, limit):
    got, ref = got.double().cpu(), ref.double()
    assert bool(torch.isfinite(got).all())
    assert float((got - ref).abs().max()) <= limit * float(ref.abs().max())


# ---------------------------------------------------------------------------------- the operators together
@pytest.mark.parametrize("dtype", [INT4, E4M3, BF16])
@pytest.mark.parametrize("heads,kv_heads,d,window,sinks", [(4, 2, 64, 0, 0), (8, 1, 128, 100, 5), (3, 3, 32, 40, 0)])
def test_chunks_through_the_cache(dtype, heads, kv_heads, d, window, sinks):
    """Three chunks of ragged conversations: each is appended, all that the cache holds is read back, and the chunk attends to
    it; then the newest token alone by `attend`, which is the chunk's last row. The reference attends to the rows read back."""
    batch, page, chunks = 3, 32, [[70, 0, 5], [1, 130, 64], [33, 2, 0]]
    total = [sum(c[b] for c in chunks) for b in range(batch)]
    pages = [-(-n // page) for n in total]
    at = _starts(pages)
    table = torch.full((batch, max(pages)), -1, dtype=torch.int32)
    for b in range(batch):
        table[b, :pages[b]] = torch.arange(at[b], at[b + 1]).flip(0)
    table = table.cuda()
    cache = serving.KVCache.allocate(at[-1], kv_heads, d, page, dtype)
    turn = rotary_table(512, d)
    past = [0] * batch
    for i, new in enumerate(chunks):
        qkv = _randn(10 * i + d, sum(new), (heads + 2 * kv_heads) * d).cuda()
        held = [p + n for p, n in zip(past, new)]
        q_at, kv_at = _starts(new), _starts(held)
        q = cache.append(qkv, heads, _i32(q_at[:-1]), _i32(new), _i32(past), table, max(new), table=turn)
        k, v = (torch.empty(kv_at[-1], kv_heads * d, dtype=BF16, device="cuda") for _ in range(2))
        cache.read(_i32(kv_at[:-1]), _i32(held), _i32([0] * batch), table, max(held), k_out=k, v_out=v)
        out = serving.packed_attention(q, k, v, _i32(q_at), _i32(kv_at), d, window=window, sinks=sinks)
        q64, k64, v64 = (x.cpu().double().view(x.shape[0], -1, d) for x in (q, k, v))
        got = out.cpu().double().view(-1, heads, d)
        for b in range(batch):
            seen = serving_fp64.visible_keys(torch.arange(past[b], held[b]), held[b], window, sinks)
            rows, keys = slice(q_at[b], q_at[b + 1]), slice(kv_at[b], kv_at[b + 1])
            for h in range(heads):
                g = h * kv_heads // heads
                ref, absum, size = serving_fp64.attend(q64[rows, h], k64[keys, g], v64[keys, g], seen, d**-0.5)
                bound = 2**-8 * ref.abs() + (2**-8 + 2**-12 + 2 * d * 2**-23 * size) * absum
                assert bool(((got[rows, h] - ref).abs() <= bound).all())
        last = [q_at[b + 1] - 1 for b in range(batch) if new[b]]
        some = [b for b in range(batch) if new[b]]
        one = cache.attend(q[last], table[some], _i32([held[b] for b in some]), window=window, sinks=sinks)
        # The two see keys and values that differ by their rounding to bf16 (half a step, 2^-8, of each product's two sides),
        # and weights of either type.
        assert float((one.double() - out[last].double()).abs().max()) <= 2**-5 * float(v64.abs().max())
        past = held


# ---------------------------------------------------------------------------------- StreamingTransformer.extend
def _model(d_model, heads, layers=2):
    cfg = TransformerConfig(3, 64, d_model, heads, 4 * d_model, layers, True)
    state = reference_fp32.round_state_to_bf16(reference_fp32.build_reference_state(cfg, 0))
    model = UserOptimizedTransformer(cfg)
    model.load_state_dict(state, strict=True)
    return model.to(device="cuda", dtype=BF16).eval(), state


CASES = [
    # d_model, heads, rotary_dim, interleaved, window, sinks, dtype, page_size
    (256, 4, 0, False, 0, 0, BF16, 16),
    (256, 4, 64, False, 0, 0, E4M3, 64),
    (256, 4, 64, False, 0, 0, INT4, 64),
    (256, 2, 128, True, 24, 4, INT4, 32),
    (256, 2, 64, False, 24, 4, BF16, 16),
    (128, 4, 32, True, 40, 0, INT4, 16),
]


@pytest.mark.parametrize("d,heads,rotary_dim,interleaved,window,sinks,dtype,page", CASES)
@torch.inference_mode()
def test_prompts_chunks_and_steps(d, heads, rotary_dim, interleaved, window, sinks, dtype, page):
    model, state = _model(d, heads)
    table = rotary_table(300, rotary_dim) if rotary_dim else None
    stream = StreamingTransformer(model, 3, 260, table=table, interleaved=interleaved, window=window, sinks=sinks, page_size=page,
                                  dtype=dtype)
    plan = [("prompt", [40, 1, 0]), ("extend", [0, 70, 33]), ("step", [2, 2, 2]), ("extend", [100, 1, 0]), ("step", [1, 1, 1]),
            ("extend", [3, 0, 0])]
    tokens = [_randn(b, sum(n[b] for _, n in plan), d) for b in range(3)]
    outs, at = [[] for _ in range(3)], [0] * 3
    for what, n in plan:
        x = [tokens[b][at[b]:at[b] + n[b]] for b in range(3)]
        if what == "prompt":
            padded = torch.zeros(3, max(n), d, dtype=BF16)
            for b in range(3):
                padded[b, :n[b]] = x[b]
            y = stream.prompt(padded.cuda(), n)
            parts = [y[b, :n[b]] for b in range(3)]
        elif what == "step":
            parts = list(stream.step(torch.stack(x).cuda()))
        else:
            parts = list(stream.extend(torch.cat(x).cuda(), n).split(n))
        for b in range(3):
            outs[b].append(parts[b])
            at[b] += n[b]
        assert stream.lengths == at
    stream.check_device_status()
    limit = {BF16: 2**-7, E4M3: 2**-4, INT4: 2**-3}[dtype]
    for b in range(3):
        ref = serving_fp64.stack(state, heads, 2, tokens[b].double(), table.cpu() if rotary_dim else None, rotary_dim, interleaved,
                                 window, sinks)
        _gate(torch.cat(outs[b]), ref, limit)


@pytest.mark.parametrize("dtype", [INT4, E4M3, BF16])
@torch.inference_mode()
def test_a_chunk_is_its_tokens_one_by_one(dtype):
    """The same codes lie in the cache either way (8-bit pages' scales grow as tokens come, so their codes may be rounded
    twice), and the outputs differ by the roundings of keys and values to bf16 and of the weights."""
    model, _ = _model(256, 4)
    table = rotary_table(128, 64)
    first, more = _randn(1, 2, 30, 256).cuda(), _randn(2, 2, 20, 256).cuda()
    streams = [StreamingTransformer(model, 2, 100, table=table, dtype=dtype) for _ in range(2)]
    for s in streams:
        s.prompt(first, [30, 11])
    chunk = streams[0].extend(more.flatten(0, 1), [20, 20]).view(2, 20, 256)
    steps = torch.cat([streams[1].step(more[:, i:i + 1]) for i in range(20)], 1)
    assert streams[0].lengths == streams[1].lengths == [50, 31]
    if dtype == BF16:
        _gate(chunk, steps.cpu(), 2**-7)
    else:
        _gate(chunk, steps.cpu(), 2**-4)


@torch.inference_mode()
def test_packed_prompts_of_fresh_sequences_are_the_models_forward():
    """Without positions and a window, over a bf16 cache."""
    model, _ = _model(256, 2)
    lengths = [150, 7, 64]
    stream = StreamingTransformer(model, 3, 150, dtype=BF16)
    x = _randn(5, 3, 150, 256).cuda()
    y = stream.extend(torch.cat([x[b, :n] for b, n in enumerate(lengths)]), lengths)
    mask = torch.arange(150, device="cuda")[None] < torch.tensor(lengths, device="cuda")[:, None]
    ref = torch.cat([r[:n] for r, n in zip(model(x, mask), lengths)])
    _gate(y, ref.cpu(), 2**-7)


@pytest.mark.parametrize("sinks,dtype", [(0, BF16), (5, E4M3), (40, INT4)])
@torch.inference_mode()
def test_a_chunk_behind_a_window_reads_what_it_sees(sinks, dtype):
    """Pages between the sinks and the band of a chunk's first token need not be there: the outputs stay as they are."""
    model, _ = _model(256, 4)
    x, more = _randn(8, 430, 256).cuda(), _randn(9, 41, 256).cuda()
    outs = []
    for gone in (False, True):
        stream = StreamingTransformer(model, 2, 480, window=33, sinks=sinks, page_size=16, dtype=dtype)
        stream.extend(x, [400, 30])
        if gone:  # the band of token 400 begins at 368; of the other sequence, at 30, everything is seen
            stream.page_table[0, -(-sinks // 16):368 // 16] = -1
        outs.append(stream.extend(more, [40, 1]))
        stream.check_device_status()
    assert torch.equal(outs[0], outs[1])


@torch.no_grad()
def test_extend_sees_changed_weights_and_any_autograd_mode():
    model, _ = _model(256, 4)
    x = _randn(3, 50, 256).cuda()

    def talk(mode):
        stream = StreamingTransformer(model, 2, 100, window=30, sinks=2, dtype=INT4)
        with torch.inference_mode(mode):
            return [stream.extend(x[:40], [25, 15]), stream.step(x[:2].view(2, 1, 256)), stream.extend(x[40:], [0, 10])]

    want = talk(False)
    for a, b in zip(talk(True), want):
        assert torch.equal(a, b)
    stream = StreamingTransformer(model, 2, 100, window=30, sinks=2, dtype=INT4)
    stream.extend(x[:40], [25, 15])
    model.layers[0].attention.q_proj.weight.mul_(0.5)
    changed = stream.extend(x[40:], [5, 5])
    fresh = StreamingTransformer(model, 2, 100, window=30, sinks=2, dtype=INT4)
    fresh.caches, fresh.lengths = stream.caches, [25, 15]
    fresh.past.copy_(_i32([25, 15]))
    assert torch.equal(fresh.extend(x[40:], [5, 5]), changed)
    y = x[:3].clone().requires_grad_()
    assert not stream.extend(y, [3, 0]).requires_grad


@torch.inference_mode()
def test_extend_refusals():
    model, _ = _model(256, 4)
    stream = StreamingTransformer(model, 2, 20, dtype=INT4)
    x = _randn(0, 12, 256).cuda()
    for bad, lengths in ((x, [12]), (x, [13, -1]), (x, [5, 5]), (x.view(2, 6, 256), [6, 6]), (x[:, :128], [6, 6]), (x.float(), [6, 6]),
                         (x.cpu(), [6, 6])):
        with pytest.raises((ValueError, RuntimeError)):
            stream.extend(bad, lengths)
    assert stream.extend(x[:0], [0, 0]).shape == (0, 256) and stream.lengths == [0, 0]
    stream.extend(x, [12, 0])
    with pytest.raises(ValueError, match="fit"):
        stream.extend(x, [12, 0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            stream.extend(x[:4], [4, 0])
        x.add(1)
    assert stream.lengths == [12, 0]
