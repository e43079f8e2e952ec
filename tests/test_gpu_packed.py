"""Attention of packed sequences on a B200, against 64-bit restatements.

Tolerances: outputs are bf16 (2^-8 of the value), weights are rounded to bf16 (2^-8), at head_dim 128 one in four exponentials is
a polynomial (2^-12), a score is a sum of head_dim fp32 products, off by at most head_dim * 2^-23 of sum |q k|, and moves a
weight by as much twice (weight and sum).
"""

import math

import pytest
import torch

from oracle import serving_fp64 as oracle
from tiktoktechjam2026track3_b200 import _capi, serving

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _clean_status(cuda_device):
    _capi.device_status(clear=True)
    yield
    torch.cuda.synchronize()
    assert _capi.device_status(clear=True) == 0


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _close(got, ref, bound):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    off = (got - ref).abs() - bound
    assert not bool((off > 0).any()), f"{float(off.nan_to_num().max())} above the bound"


def _starts(lengths, first=0):
    at = [first]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def _check(q, k, v, out, q_at, kv_at, heads, kv_heads, d, window, sinks, rows=None):
    q, k, v = (x.cpu().double().reshape(x.shape[0], -1, d) for x in (q, k, v))
    got = out.cpu().reshape(out.shape[0], heads, d)
    for b in range(len(q_at) - 1):
        n_q, n = q_at[b + 1] - q_at[b], kv_at[b + 1] - kv_at[b]
        some = torch.arange(n_q) if rows is None else torch.tensor([r for r in rows if r < n_q], dtype=torch.long)
        seen = oracle.visible_keys(n - n_q + some, n, window, sinks)
        for h in range(heads):
            kv = h * kv_heads // heads
            ref, absum, size = oracle.attend(q[q_at[b] + some, h], k[kv_at[b]:kv_at[b + 1], kv], v[kv_at[b]:kv_at[b + 1], kv], seen,
                                             d**-0.5)
            _close(got[q_at[b] + some, h], ref, 2**-8 * ref.abs() + (2**-8 + 2**-12 + 2 * d * 2**-23 * size) * absum)


CASES = [
    # queries, keys before them (None: whole prompts), heads, kv_heads, head_dim, window, sinks
    ([1], None, 1, 1, 64, 0, 0),
    ([5, 130, 1, 0, 64], None, 4, 4, 64, 0, 0),
    ([128, 256, 127, 129], None, 2, 1, 128, 0, 0),
    ([300, 0, 0, 17], None, 6, 2, 32, 0, 0),             # a group of three: no packing of heads
    ([70, 200], None, 16, 1, 64, 0, 0),                  # sixteen heads to a tile
    ([33, 90], None, 32, 1, 32, 0, 0),                   # thirty-two: two tiles of sixteen
    ([40, 7, 150], [300, 0, 1], 8, 2, 64, 0, 0),
    ([64, 1, 129], [1000, 129, 0], 4, 4, 128, 0, 0),
    ([1, 2, 3, 1], [0, 500, 127, 128], 12, 2, 128, 0, 0),
    ([200, 400], None, 4, 2, 64, 100, 4),
    ([90, 33, 260], [700, 5, 131], 4, 2, 128, 64, 20),
    ([300, 20], [40, 600], 2, 2, 32, 130, 131),          # sinks over more than a tile, not a multiple of 16
    ([500], [300], 1, 1, 128, 300, 600),                 # sinks beyond the window
    ([77, 78], [10, 200], 3, 3, 64, 1, 0),               # a window of the token itself
    ([60, 10], [100, 3000], 5, 1, 64, 100000, 7),        # a window longer than everything
    ([3] * 70 + [130], None, 2, 2, 64, 0, 0),            # more sequences than one turn of the search takes
]


@pytest.mark.parametrize("new,past,heads,kv_heads,d,window,sinks", CASES)
@pytest.mark.parametrize("junk", [False, True])
def test_packed_attention(new, past, heads, kv_heads, d, window, sinks, junk):
    """Column slices of packed projections, or q apart from k and v; with `junk`, rows before the first and behind the last
    sequence hold NaN, and stay as they are in the output."""
    g = _gen(sum(new) + heads)
    first, behind = (3, 40) if junk else (0, 0)
    q_at = _starts(new, first)
    kv_at = q_at if past is None else _starts([n + p for n, p in zip(new, past)], first)
    width = (heads + 2 * kv_heads) * d
    packed = torch.randn(max(q_at[-1], kv_at[-1]) + behind, width + 8, generator=g).bfloat16()
    packed[:first] = math.nan
    if junk:
        packed[kv_at[-1]:] = math.nan
    packed = packed.cuda()
    k, v = packed[:, heads * d:(heads + kv_heads) * d], packed[:, (heads + kv_heads) * d:width]
    q = packed[:, :heads * d][:q_at[-1] + behind]
    out = torch.full((q.shape[0], heads * d + 16), 3.0, dtype=BF16, device="cuda")
    got = serving.packed_attention(q, k, v, _i32(q_at), None if past is None else _i32(kv_at), d, window=window, sinks=sinks,
                                   out=out[:, 8:8 + heads * d])
    _check(q, k, v, got, q_at, kv_at, heads, kv_heads, d, window, sinks)
    assert bool((out[:first] == 3.0).all()) and bool((out[q_at[-1]:] == 3.0).all())
    assert bool((out[:, :8] == 3.0).all()) and bool((out[:, 8 + heads * d:] == 3.0).all())
    fresh = serving.packed_attention(q, k, v, _i32(q_at), _i32(kv_at), d, window=window, sinks=sinks)
    assert torch.equal(fresh[first:q_at[-1]], got[first:q_at[-1]])
    assert not bool(fresh[:first].any()) and not bool(fresh[q_at[-1]:].any())


@pytest.mark.parametrize("heads,kv_heads,d", [(2, 2, 64), (4, 1, 128), (16, 1, 32)])
def test_more_queries_than_keys_and_no_keys(heads, kv_heads, d):
    """Queries before the first key see nothing: zeros, whole tiles of them too, and where there are no keys at all."""
    new, keys = [200, 5, 300, 40], [50, 0, 0, 39]
    q_at, kv_at = _starts(new), _starts(keys)
    g = _gen(1)
    q = torch.randn(q_at[-1], heads * d, generator=g).bfloat16().cuda()
    k, v = (torch.randn(kv_at[-1], kv_heads * d, generator=g).bfloat16().cuda() for _ in range(2))
    for window, sinks in ((0, 0), (20, 3)):
        out = torch.full_like(q, 9.0)
        serving.packed_attention(q, k, v, _i32(q_at), _i32(kv_at), d, window=window, sinks=sinks, out=out)
        _check(q, k, v, out, q_at, kv_at, heads, kv_heads, d, window, sinks)
        assert not bool(out[:150].any()) and not bool(out[200:505].any())
    none = serving.packed_attention(q, k[:0], v[:0], _i32(q_at), _i32([0] * 5), d)
    assert not bool(none.any())


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 4), (50, 130)])
def test_a_sequence_does_not_see_its_neighbours(d, window, sinks):
    """Every other sequence holds NaN and infinities in queries, keys and values: the others' results are the same bits
    as by themselves."""
    heads, kv_heads, new, past = 4, 2, [40, 170, 1, 129, 300], [7, 100, 60, 0, 130]
    q_at, kv_at = _starts(new), _starts([n + p for n, p in zip(new, past)])
    g = _gen(d)
    q = torch.randn(q_at[-1], heads * d, generator=g).bfloat16()
    k, v = (torch.randn(kv_at[-1], kv_heads * d, generator=g).bfloat16() for _ in range(2))
    for b in (0, 2, 4):
        q[q_at[b]:q_at[b + 1]] = math.nan
        k[kv_at[b]:kv_at[b + 1]] = math.inf
        v[kv_at[b]:kv_at[b + 1]] = math.nan
    q, k, v = q.cuda(), k.cuda(), v.cuda()
    out = serving.packed_attention(q, k, v, _i32(q_at), _i32(kv_at), d, window=window, sinks=sinks)
    for b in (1, 3):
        own = serving.packed_attention(q[q_at[b]:q_at[b + 1]], k[kv_at[b]:kv_at[b + 1]], v[kv_at[b]:kv_at[b + 1]],
                                       _i32([0, new[b]]), _i32([0, new[b] + past[b]]), d, window=window, sinks=sinks)
        assert bool(torch.isfinite(own).all())
        assert torch.equal(out[q_at[b]:q_at[b + 1]], own)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,window,sinks,at", [
    (2, 2, 100, 4, [4, 5, 15]), (4, 1, 33, 20, [20, 31]), (2, 1, 64, 130, [130, 143]), (16, 1, 50, 1, [1, 15])])
def test_values_behind_the_sinks_reach_only_the_rows_near_those_that_see_them(d, heads, kv_heads, window, sinks, at):
    n, first = 700, 37
    g = _gen(d + sinks)
    q = torch.randn(first + n, heads * d, generator=g).bfloat16()
    k, v = (torch.randn(first + n, kv_heads * d, generator=g).bfloat16() for _ in range(2))
    for i, j in enumerate(at):
        v[first + j] = (math.nan, math.inf, -math.inf)[i]
    out = serving.packed_attention(q.cuda(), k.cuda(), v.cuda(), _i32([0, first, first + n]), None, d, window=window, sinks=sinks)
    out = out.cpu().view(first + n, heads, d)[first:]
    rows = torch.cat([torch.arange(min(at) // 128 * 128), torch.arange(max(at) + window + 127, n)])
    seen = oracle.visible_keys(rows, n, window, sinks)
    assert not bool(seen[:, at].any())
    q, k, v = (x.double().view(first + n, -1, d)[first:] for x in (q, k, v))
    v[at] = 0.0
    for h in range(heads):
        kv = h * kv_heads // heads
        ref, absum, size = oracle.attend(q[rows, h], k[:, kv], v[:, kv], seen, d**-0.5)
        _close(out[rows, h], ref, 2**-8 * ref.abs() + (2**-8 + 2**-12 + 2 * d * 2**-23 * size) * absum)


@pytest.mark.parametrize("d,window,sinks", [(32, 0, 0), (64, 0, 0), (128, 0, 0), (64, 150, 16), (128, 150, 16)])
def test_whole_prompts_are_the_window_attention(d, window, sinks):
    """Packed sequences of one length are the padded batch's, bit for bit (sinks a multiple of 16)."""
    batch, seq, heads, kv_heads = 3, 333, 4, 2
    qkv = torch.randn(batch * seq, (heads + 2 * kv_heads) * d, generator=_gen(d)).bfloat16().cuda()
    q, k, v = qkv.split([heads * d, kv_heads * d, kv_heads * d], 1)
    out = serving.packed_attention(q, k, v, _i32([seq * b for b in range(batch + 1)]), None, d, window=window, sinks=sinks)
    assert torch.equal(out, serving.window_attention(q, k, v, batch, seq, d, window=window, sinks=sinks))


def test_long_chunk_behind_a_long_cache():
    """Far positions, the head-major order: some rows of a chunk of 3000 behind 40000 keys."""
    d, heads, kv_heads, new, past = 64, 4, 1, [10, 3000], [3, 40000]
    q_at, kv_at = _starts(new), _starts([n + p for n, p in zip(new, past)])
    g = _gen(2)
    q = torch.randn(q_at[-1], heads * d, generator=g).bfloat16().cuda()
    k, v = (torch.randn(kv_at[-1], kv_heads * d, generator=g).bfloat16().cuda() for _ in range(2))
    for window, sinks in ((0, 0), (2500, 7)):
        out = serving.packed_attention(q, k, v, _i32(q_at), _i32(kv_at), d, window=window, sinks=sinks)
        _check(q, k, v, out, q_at, kv_at, heads, kv_heads, d, window, sinks, rows=[0, 9, 31, 1234, 2968, 2999])


@pytest.mark.parametrize("q_at,kv_at", [([0, 10, 5, 20], [0, 10, 5, 20]), ([0, 10, 50], [0, 10, 20]), ([0, 10, 20], [0, 10, 50]),
                                        ([-3, 10, 20], [0, 10, 20]), ([0, 10, 20], [0, 30, 20]), ([5, -1, 4], [0, 5, 10])])
def test_sequences_outside_the_rows_are_skipped_and_recorded(q_at, kv_at):
    q, k, v = (torch.randn(20, 64, generator=_gen(i)).bfloat16().cuda() for i in range(3))
    out = torch.full_like(q, 5.0)
    serving.packed_attention(q, k, v, _i32(q_at), _i32(kv_at), 64, out=out)
    torch.cuda.synchronize()
    assert _capi.device_status(clear=True) == (9 << 16) | (1 << 8) | 3
    for b in range(len(q_at) - 1):
        if 0 <= q_at[b] <= q_at[b + 1] <= 20 and 0 <= kv_at[b] <= kv_at[b + 1] <= 20 and q_at == sorted(q_at):
            _check(q, k, v, out, q_at[b:b + 2], kv_at[b:b + 2], 1, 1, 64, 0, 0)
            out[q_at[b]:q_at[b + 1]] = 5.0
    if q_at == sorted(q_at):
        assert bool((out == 5.0).all())
