"""The serving operators where calls, memory and odd values meet, on a B200, against 64-bit restatements.

Tolerances are those of test_gpu_serving.py, by the same arithmetic.
"""

import math

import pytest
import torch

from oracle import serving_fp64 as oracle
from test_gpu_serving import _check_attend, _close, _filled, _gen, _i32
from tiktoktechjam2026track3_b200 import TransformerConfig, UserOptimizedTransformer, _capi, serving

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
    more = torch.randn(16, 8 * 64, generator=_gen(4)).bfloat16().cuda()  # four tokens each: a larger workspace
    want, larger = cache.attend(q[:1], table[:1], n[:1]), cache.attend(more, table, n, q_len=4)
    out = torch.empty_like(q[:1])
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.attend(q[:1], table[:1], n[:1], out=out)
        with torch.cuda.graph(graph, stream=side):
            cache.attend(q[:1], table[:1], n[:1], out=out)
        assert torch.equal(cache.attend(more, table, n, q_len=4), larger)
        others = [torch.full((1 << 20,), 7, dtype=torch.uint8, device="cuda") for _ in range(40)]
        out.zero_()
        graph.replay()
        again = cache.attend(more, table, n, q_len=4)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(again, larger)
    assert all(bool((x == 7).all()) for x in others)


@pytest.mark.parametrize("heads", [1, 8])
@pytest.mark.parametrize("room", [0, 1 << 17])
def test_steps_enqueued_at_once_are_those_waited_for_one_by_one(heads, room):
    """Append and attend in turn without a wait between, with magnitudes that make the page's scale grow every few
    steps (neighbouring heads' scales lie in one sector): the same bits as with a wait after every call."""
    steps, d = 40, 64
    g = _gen(11)
    grow = torch.exp2(torch.arange(steps) / 3.0)[:, None]
    rows = (torch.randn(steps, 3 * heads * d, generator=g) * grow).bfloat16().cuda()
    got = []
    for wait in (False, True):
        cache = serving.KVCache.allocate(4, heads, d, 16)
        table = torch.nn.functional.pad(_i32([[2, 0, 3]]), (0, max(0, room // 16 - 3)), value=-1)
        past, lens = [_i32([i]) for i in range(steps)], [_i32([i + 1]) for i in range(steps)]
        zero, one = _i32([0]), _i32([1])
        torch.cuda.synchronize()
        outs = []
        for i in range(steps):
            cache.append(rows[i:i + 1], heads, zero, one, past[i], table, 1)
            if wait:
                torch.cuda.synchronize()
            outs.append(cache.attend(rows[i:i + 1, :heads * d], table, lens[i]))
            if wait:
                torch.cuda.synchronize()
        got.append(torch.cat(outs))
    assert torch.equal(*got)


@pytest.mark.parametrize("heads,kv_heads,head_dim,q_len,dtype", [
    (16, 1, 64, 5, E4M3), (40, 2, 128, 27, BF16), (12, 1, 32, 47, E4M3), (16, 2, 128, 65, E4M3)])
def test_attend_with_more_row_blocks_than_one_launch_takes(heads, kv_heads, head_dim, q_len, dtype):
    lengths = [1100, 30, 3000]
    cache, seqs = _filled(lengths, 64, kv_heads, head_dim, dtype, 8)
    q = torch.randn(len(lengths) * q_len, heads * head_dim, generator=_gen(2)).bfloat16().cuda()
    outs = [cache.attend(q, table, _i32(lengths), q_len=q_len) for table in (seqs.table.cuda(), _wide(seqs, 64)) for _ in range(2)]
    for out in outs[::2]:
        _check_attend(cache, seqs, lengths, heads, q_len, 0, 0, q, out, head_dim**-0.5)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[2], outs[3])


def test_one_workspace_for_calls_of_any_shape():
    """Many newest tokens of one sequence, then one of many, on different caches, through one workspace of the caller's."""
    lengths = [4000] + [70 + 5 * b for b in range(63)]
    caches = [_filled(lengths, 64, 2, 64, E4M3, 1), _filled(lengths, 64, 1, 128, BF16, 2)]
    calls = []
    for cache, seqs in caches:
        table = _wide(seqs, 64)
        for batch, q_len in ((1, 16), (64, 1), (3, 4), (64, 2), (1, 1)):
            q = torch.randn(batch * q_len, 4 * cache.head_dim, generator=_gen(batch)).bfloat16().cuda()
            args = (q, table[:batch], _i32(lengths[:batch]))
            fresh = cache.workspace(batch, 4, q_len)
            calls.append((cache, args, q_len, cache.attend(*args, q_len=q_len, workspace=fresh)))
    shared = max((c.workspace(1, 4, 16) for c, _ in caches), key=lambda w: w.numel())
    for order in (calls, calls[::-1], calls[::2] + calls[1::2]):
        for cache, args, q_len, want in order:
            assert torch.equal(cache.attend(*args, q_len=q_len, workspace=shared), want)
    _check_attend(*caches[0], lengths, 4, 1, 0, 0, calls[1][1][0], calls[1][3], 64**-0.5)


# ---------------------------------------------------------------------------------- values that are not finite
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,window,sinks,at", [
    (2, 2, 100, 4, [4, 5, 15]), (4, 1, 33, 20, [20, 31]), (2, 1, 64, 130, [130, 143]), (1, 1, 100, 4, [16, 17]),
    (16, 1, 50, 1, [1, 15]), (3, 3, 40, 270, [271])])
def test_values_behind_the_sinks_reach_only_the_rows_near_those_that_see_them(d, heads, kv_heads, window, sinks, at):
    """Infinities and NaN in the values of tokens right behind the sinks: at most the rows less than 128 from one that
    sees them may be touched (the tokens lie in the same 16 rows as the last sink, which every later row sees)."""
    n = 900
    g = _gen(d + sinks)
    q = torch.randn(n, heads * d, generator=g).bfloat16()
    k, v = (torch.randn(n, kv_heads * d, generator=g).bfloat16() for _ in range(2))
    for i, j in enumerate(at):
        v[j] = (math.nan, math.inf, -math.inf)[i]
    out = serving.window_attention(q.cuda(), k.cuda(), v.cuda(), 1, n, d, window=window, sinks=sinks).cpu().view(n, heads, d)
    rows = torch.cat([torch.arange(min(at) // 128 * 128), torch.arange(max(at) + window + 127, n)])
    seen = oracle.visible_keys(rows, n, window, sinks)
    assert not bool(seen[:, at].any())
    q, k, v = (x.double().view(n, -1, d) for x in (q, k, v))
    v[at] = 0.0
    for h in range(heads):
        kv = h * kv_heads // heads
        ref, absum, size = oracle.attend(q[rows, h], k[:, kv], v[:, kv], seen, d**-0.5)
        _close(out[rows, h], ref, 2**-8 * ref.abs() + (2**-8 + 2**-12 + 2 * d * 2**-23 * size) * absum)


@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("heads,kv_heads,head_dim,page,lengths", [
    (4, 2, 32, 16, [1, 17, 33, 500]), (3, 3, 64, 32, [16, 49, 1000]), (20, 2, 32, 64, [5, 130]), (8, 1, 128, 16, [47]),
    (1, 1, 64, 16, [0, 3])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
@pytest.mark.parametrize("room", [0, 1 << 17])
def test_scales_of_pages_that_no_row_sees_are_not_used(junk, heads, kv_heads, head_dim, page, lengths, window, sinks, room):
    """Scales as an allocation leaves them in pages that nobody owns, page 0 among them (tiles that are missing at a
    sequence's end read it)."""
    cache, seqs = _filled(lengths, page, kv_heads, head_dim, E4M3, 6)
    last = seqs.pages - 1
    used = sorted(int(i) for i in seqs.table.flatten() if i >= 0)
    if 0 in used:  # the owner of page 0 takes an unused page instead
        free = next(i for i in range(last, 0, -1) if i not in used)
        for x in (cache.k, cache.v):
            x.view(torch.uint8)[free] = x.view(torch.uint8)[0]
            x.view(torch.uint8)[0] = 0x7f  # the code of a NaN
        for x in (cache.k_scale, cache.v_scale):
            x[free] = x[0]
        seqs.table[seqs.table == 0] = free
        used[used.index(0)] = free
    unowned = [i for i in range(seqs.pages) if i not in used]
    assert 0 in unowned
    cache.k_scale[unowned] = junk
    cache.v_scale[unowned] = junk
    table = _wide(seqs, page, room) if room else seqs.table.cuda()
    q = torch.randn(len(lengths), heads * head_dim, generator=_gen(1)).bfloat16().cuda()
    out = cache.attend(q, table, _i32(lengths), window=window, sinks=sinks)
    kept = serving.KVCache(cache.k, cache.v, cache.k_scale.nan_to_num(1.0, 1.0, 1.0), cache.v_scale.nan_to_num(1.0, 1.0, 1.0))
    _check_attend(kept, seqs, lengths, heads, 1, window, sinks, q, out, head_dim**-0.5)


# ---------------------------------------------------------------------------------- wrong indices
def test_a_wrong_index_does_not_stop_other_callers():
    """One caller's position past its table is reported to those who ask for indices; a model's forward goes on."""
    model = UserOptimizedTransformer(TransformerConfig(1, 16, 64, 1, 64, 1, True)).to("cuda", BF16).eval()
    x = torch.randn(1, 16, 64, generator=_gen(1)).bfloat16().cuda()
    rows = torch.randn(2, 64, generator=_gen(2)).bfloat16().cuda()
    watch = _capi.StatusWatch(indices=True)
    with torch.inference_mode():
        before = model(x)
        model.check_device_status()
        serving.rotary(rows, _i32([0, 16]), serving.rotary_table(16, 64), 64)
        after = model(x)
        model.check_device_status()
        assert torch.equal(model(x), before) and torch.equal(after, before)
        model.check_device_status()
    watch.after_forward(rows.device)
    with pytest.raises(RuntimeError, match="rotary kernel met an index outside its table.*skipped"):
        watch.check(wait=True)
    assert _capi.device_status(clear=True) == (5 << 16) | (1 << 8) | 3
    watch.after_forward(rows.device)
    assert watch.check(wait=True) == 0
