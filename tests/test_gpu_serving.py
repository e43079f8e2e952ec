"""Rotary positions, the paged cache and the attention over it, on a B200, against 64-bit restatements.

Tolerances follow from the arithmetic: outputs are bf16 (half an ulp is at most 2^-8 of a power of two below the
value, so 2^-9 of the next one: |error| <= 2^-8 |y| covers it with the rest of its bound), products and sums are fp32.
Attention weights are rounded to fp16 (2^-11 relative) over an 8-bit cache and to bf16 (2^-8) over a bf16
one, which moves the output by at most that share of sum_j w_j |v_j|; a score is a sum of head_dim fp32
products, off by at most head_dim * 2^-23 of sum |q k|, and moves weights by as much, relatively, twice (weight and sum).
"""

import math

import pytest
import torch

from oracle import serving_fp64 as oracle
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


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _close(got, ref, bound):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    off = (got - ref).abs() - bound
    assert not bool((off > 0).any()), f"{float(off.nan_to_num().max())} above the bound"


# ---------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("tokens,heads,head_dim,rotary_dim", [
    (1, 1, 16, 16), (1, 24, 64, 64), (77, 3, 128, 128), (513, 5, 128, 48), (9, 40, 256, 240), (300, 1, 48, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary(tokens, heads, head_dim, rotary_dim, interleaved, inverse):
    g = _gen(tokens + head_dim)
    table = serving.rotary_table(2000, rotary_dim)
    packed = torch.randn(tokens, heads * head_dim + 24, generator=g).bfloat16().cuda()
    x = packed[:, 8:8 + heads * head_dim]  # a column slice: row stride above the width
    pos = torch.randint(0, 2000, (tokens,), generator=g, dtype=torch.int32)
    y = serving.rotary(x, pos.cuda(), table, head_dim, interleaved=interleaved, inverse=inverse)
    x64 = x.cpu().view(tokens, heads, head_dim)
    ref = oracle.rotate(x64, table.cpu()[pos.long()], rotary_dim, interleaved, inverse)
    size = x64.abs().amax(-1, keepdim=True).double()
    _close(y.view(tokens, heads, head_dim), ref, 2**-8 * ref.abs() + 2**-22 * size)
    if head_dim > rotary_dim:
        assert torch.equal(y.view(tokens, heads, head_dim)[..., rotary_dim:].cpu(), x64[..., rotary_dim:])
    serving.rotary(x, pos.cuda(), table, head_dim, out=x, interleaved=interleaved, inverse=inverse)
    assert torch.equal(x, y)  # in place


def test_rotary_gradient_against_differences():
    """inverse=True is the transpose: <g, R x> = <R^T g, x>, and each partial derivative of <g, R x> by differences."""
    g = _gen(5)
    table = serving.rotary_table(64, 32)
    for interleaved in (False, True):
        x = torch.randn(4, 64, generator=g)
        grad_out = torch.randn(4, 64, generator=g).bfloat16()
        pos = torch.tensor([0, 1, 17, 63], dtype=torch.int32)
        grad = serving.rotary(grad_out.cuda(), pos.cuda(), table, 32, interleaved=interleaved, inverse=True).cpu()

        def value(z):
            y = oracle.rotate(z.view(4, 2, 32), table.cpu()[pos.long()], 32, interleaved)
            return (y.view(4, 64) * grad_out.double()).sum(-1)

        step = 0.5  # the function is linear: any step is exact
        for c in range(0, 64, 7):
            d = torch.zeros(4, 64, dtype=torch.float64)
            d[:, c] = step
            slope = (value(x.double() + d) - value(x.double() - d)) / (2 * step)
            _close(grad[:, c], slope, 2**-8 * slope.abs() + 2**-20)


def test_rotary_rows_without_a_token_and_out_of_table():
    table = serving.rotary_table(16, 32)
    x = torch.randn(4, 64, generator=_gen(1)).bfloat16().cuda()
    out = torch.full_like(x, 7.0)
    serving.rotary(x, _i32([-1, 3, 16, -5]), table, 32, out=out)
    assert bool((out[[0, 2, 3]] == 7.0).all()) and not bool((out[1] == 7.0).any())
    torch.cuda.synchronize()
    assert _capi.device_status(clear=True) == (5 << 16) | (1 << 8) | 3
    serving.rotary(x[:0], _i32([]), table, 32, out=out[:0])  # no rows: nothing to do


# ---------------------------------------------------------------------------------- append
class _Sequences:
    """Sequences with pages in random order."""

    def __init__(self, lengths, page_size, seed, spare=2):
        counts = [-(-n // page_size) for n in lengths]
        order = torch.randperm(sum(counts) + spare, generator=_gen(seed)).tolist()
        self.pages = sum(counts) + spare
        self.table = torch.full((len(lengths), max(1, max(counts))), -1, dtype=torch.int32)
        for b, n in enumerate(counts):
            for i in range(n):
                self.table[b, i] = order.pop()


def _values(cache, which):
    """The values that a cache's pages stand for, float64 on the CPU."""
    x, scale = (cache.k, cache.k_scale) if which == "k" else (cache.v, cache.v_scale)
    x = x.cpu().float().double()
    return x if scale is None else x * scale.cpu().double()[:, :, None, None]


def _gather(cache, which, table, length):
    page = cache.page_size
    ids = table[: -(-length // page)].long()
    x = _values(cache, which)[ids]  # [n, heads, page, d]
    return x.transpose(0, 1).reshape(cache.kv_heads, -1, cache.head_dim)[:, :length]


APPENDS = [
    # new, past, page_size, heads, kv_heads, head_dim, rotary_dim, interleaved
    ([1], [0], 16, 1, 1, 16, 16, False),
    ([1, 1, 1], [15, 16, 0], 16, 4, 2, 64, 64, False),
    ([5, 0, 40], [31, 7, 33], 32, 3, 3, 64, 32, True),
    ([130, 1], [0, 200], 64, 10, 2, 128, 128, False),
    ([77, 300, 3], [60, 1, 127], 128, 6, 1, 128, 48, True),
    ([17], [250], 256, 2, 2, 256, 256, False),
]


@pytest.mark.parametrize("new,past,page,heads,kv_heads,head_dim,rotary_dim,interleaved", APPENDS)
@pytest.mark.parametrize("dtype", [E4M3, BF16])
@pytest.mark.parametrize("rotated", [True, False])
def test_append(new, past, page, heads, kv_heads, head_dim, rotary_dim, interleaved, dtype, rotated):
    g = _gen(sum(new) + page)
    seqs = _Sequences([n + p for n, p in zip(new, past)], page, 3)
    cache = serving.KVCache.allocate(seqs.pages, kv_heads, head_dim, page, dtype)
    table = serving.rotary_table(2048, rotary_dim) if rotated else None
    step = dict(table=table, interleaved=interleaved)
    pages = seqs.table.cuda()

    def rows(n):
        return (torch.randn(n, (heads + 2 * kv_heads) * head_dim, generator=g) * 3).bfloat16()

    def starts(lengths):
        return [sum(lengths[:i]) for i in range(len(lengths))]

    first = rows(sum(past))  # what the cache already holds, smaller than what follows, so that scales grow
    if sum(past):
        cache.append((first * 0.25).cuda(), heads, _i32(starts(past)), _i32(past), _i32([0] * len(past)), pages,
                     max(past), **step)
    before = {w: _values(cache, w) for w in "kv"}
    scales = {"k": cache.k_scale.clone(), "v": cache.v_scale.clone()} if dtype == E4M3 else None
    qkv = rows(sum(new))
    k_out = torch.full((sum(new), kv_heads * head_dim), 9.0, dtype=BF16, device="cuda")
    q_out = cache.append(qkv.cuda(), heads, _i32(starts(new)), _i32(new), _i32(past), pages, max(new), k_out=k_out,
                         **step)
    x = qkv.double().view(-1, heads + 2 * kv_heads, head_dim)
    if rotated:
        pos = torch.cat([torch.arange(p, p + n) for n, p in zip(new, past)])
        turned = oracle.rotate(x[:, :heads + kv_heads], table.cpu()[pos], rotary_dim, interleaved)
        size = x[:, :heads + kv_heads].abs().amax(-1, keepdim=True)
        bound = 2**-8 * turned.abs() + 2**-22 * size
        _close(q_out.view(-1, heads, head_dim), turned[:, :heads], bound[:, :heads])
        _close(k_out.view(-1, kv_heads, head_dim), turned[:, heads:], bound[:, heads:])
        keys = turned[:, heads:]
    else:
        assert q_out is None
        keys = x[:, heads:heads + kv_heads]
        assert torch.equal(k_out.cpu().double().view(-1, kv_heads, head_dim), keys)
    for which, fresh in (("k", keys), ("v", x[:, heads + kv_heads:])):
        inexact = which == "k" and rotated  # 64-bit and 32-bit rotations may round to neighbouring codes
        now = _values(cache, which)
        expect = before[which].clone()
        row = 0
        for b, (n, p) in enumerate(zip(new, past)):
            at = p
            while at < p + n:
                stop = min((at // page + 1) * page, p + n)
                pid, slot = int(seqs.table[b, at // page]), at % page
                part = fresh[row:row + stop - at].transpose(0, 1)  # [heads, tokens, d]
                row += stop - at
                for h in range(kv_heads):
                    if dtype == BF16:
                        expect[pid, h, slot:slot + stop - at] = part[h]
                        continue
                    e = oracle.scale_exponent(part[h])
                    if slot:
                        e = max(e, round(math.log2(float(scales[which][pid, h]))))
                        old = before[which][pid, h, :slot]
                        expect[pid, h, :slot] = oracle.e4m3(old * 2.0**-e) * 2.0**e
                    got_e = (cache.k_scale if which == "k" else cache.v_scale)[pid, h].log2().item()
                    assert got_e == e
                    stale = before[which][pid, h, slot + stop - at:] / float(scales[which][pid, h])
                    expect[pid, h, slot + stop - at:] = stale * 2.0**e  # codes not touched
                    expect[pid, h, slot:slot + stop - at] = oracle.e4m3(part[h] * 2.0**-e) * 2.0**e
                at = stop
        if dtype == BF16:
            _close(now, expect, 2**-8 * expect.abs() + 2**-20 * 12 if inexact else 0 * expect)
        else:
            wrong = now != expect
            # A code can differ only where the exact value lies within fp32's error of a tie: a few in a million.
            assert int(wrong.sum()) <= (2 + wrong.numel() // 50000 if inexact else 0)
            _close(now, expect, 2**-3 * expect.abs() + 2**-9 if inexact else 0 * expect)


def test_append_in_place_matches_separate_outputs():
    heads, kv_heads, d = 6, 2, 64
    seqs = _Sequences([70], 32, 1)
    table = serving.rotary_table(128, d)
    qkv = torch.randn(70, (heads + 2 * kv_heads) * d, generator=_gen(2)).bfloat16().cuda()
    got = []
    for in_place in (False, True):
        cache = serving.KVCache.allocate(seqs.pages, kv_heads, d, 32)
        x = qkv.clone()
        q = x[:, :heads * d] if in_place else torch.empty(70, heads * d, dtype=BF16, device="cuda")
        k = x[:, heads * d:(heads + kv_heads) * d] if in_place else torch.empty(70, kv_heads * d, dtype=BF16, device="cuda")
        cache.append(x, heads, _i32([0]), _i32([70]), _i32([0]), seqs.table.cuda(), 70, table=table, q_out=q, k_out=k)
        got.append((q.clone(), k.clone(), cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_append_values_that_do_not_fit():
    """Infinities and NaN become the NaN code and do not set the scale; a page of zeros; magnitudes past the range."""
    cache = serving.KVCache.allocate(3, 1, 16, 16)
    qkv = torch.zeros(4, 48).bfloat16()
    qkv[0, 16:32] = 1.0
    qkv[0, 16], qkv[0, 17], qkv[0, 18] = math.inf, -math.inf, math.nan
    qkv[1, 16:32] = 896.0
    qkv[1, 32:48] = 2.0**60
    cache.append(qkv.cuda(), 1, _i32([0, 1, 2]), _i32([1, 1, 2]), _i32([0, 0, 0]), _i32([[0], [1], [2]]), 2)
    k, v = _values(cache, "k"), _values(cache, "v")
    assert bool(torch.isnan(k[0, 0, 0, :3]).all()) and bool((k[0, 0, 0, 3:] == 1.0).all())
    assert float(cache.k_scale[0, 0]) == 2.0**-8 and float(cache.k_scale[1, 0]) == 2.0
    assert bool((k[1, 0, 0] == 896.0).all())
    assert float(cache.v_scale[1, 0]) == 2.0**40 and bool((v[1, 0, 0] == 448.0 * 2.0**40).all())
    assert float(cache.k_scale[2, 0]) == 2.0**-40 and bool((k[2] == 0).all())


def test_append_indices_outside_their_tables_write_nothing():
    qkv = torch.ones(4, 48, dtype=BF16, device="cuda")
    for start, count, past, pages in ((0, 5, 0, [[0, 1]]), (2, 3, 0, [[0, 1]]), (0, 4, 30, [[0, 1]]), (0, 4, 0, [[9, 1]]),
                                      (-1, 2, 0, [[0, 1]]), (0, 4, -2, [[0, 1]]), (0, 3, 0, [[-1, -1]])):
        cache = serving.KVCache.allocate(2, 1, 16, 16)
        cache.append(qkv, 1, _i32([start]), _i32([count]), _i32([past]), _i32(pages), 4)
        torch.cuda.synchronize()
        status = _capi.device_status(clear=True)
        assert status >> 16 == 6 and status & 0xFF == 3
        assert not bool(cache.k.float().any())


# ---------------------------------------------------------------------------------- attention over the cache
def _filled(lengths, page, kv_heads, d, dtype, seed, spread=1.0, junk=math.nan):
    """A cache holding random keys and values, NaN in every slot and page that no sequence uses."""
    seqs = _Sequences(lengths, page, seed)
    g = _gen(seed)
    cache = serving.KVCache.allocate(seqs.pages, kv_heads, d, page, dtype)
    cache.k.copy_(torch.full(cache.k.shape, junk).to(dtype))
    cache.v.copy_(torch.full(cache.v.shape, junk).to(dtype))
    n = sum(lengths)
    qkv = torch.randn(n, 3 * kv_heads * d, generator=g)
    qkv *= torch.exp2(torch.randint(-3, 4, (n, 1), generator=g) * spread)  # pages of unlike magnitude
    start = [sum(lengths[:b]) for b in range(len(lengths))]
    cache.append(qkv.bfloat16().cuda(), kv_heads, _i32(start), _i32(lengths), _i32([0] * len(lengths)),
                 seqs.table.cuda(), max(lengths))
    return cache, seqs


def _check_attend(cache, seqs, lengths, heads, q_len, window, sinks, q, out, scale):
    d, hk = cache.head_dim, cache.kv_heads
    q64 = q.cpu().double().view(len(lengths), q_len, heads, d)
    got = out.cpu().view(len(lengths), q_len, heads, d)
    weight = 2**-10 if cache.quantised else 2**-8
    for b, n in enumerate(lengths):
        k, v = _gather(cache, "k", seqs.table[b], n), _gather(cache, "v", seqs.table[b], n)
        seen = oracle.visible_keys(torch.arange(n - q_len, n), n, window, sinks)
        for h in range(heads):
            ref, absum, size = oracle.attend(q64[b, :, h], k[h * hk // heads], v[h * hk // heads], seen, scale)
            _close(got[b, :, h], ref, 2**-8 * ref.abs() + (weight + 2 * d * 2**-23 * size + 2**-18) * absum)


ATTENDS = [
    # lengths, page_size, heads, kv_heads, head_dim, q_len, window, sinks
    ([1], 16, 1, 1, 64, 1, 0, 0),
    ([0, 5, 16, 17], 16, 2, 1, 32, 1, 0, 0),
    ([100, 1000, 31], 16, 12, 12, 64, 1, 0, 0),
    ([257, 64], 64, 10, 2, 128, 1, 0, 0),
    ([2000], 128, 16, 1, 128, 1, 0, 0),          # 16 query heads of one key head: one block of 16 rows
    ([700, 3], 32, 20, 1, 64, 1, 0, 0),          # 20: two blocks
    ([500, 130, 2], 16, 6, 2, 128, 3, 0, 0),     # drafts; a sequence shorter than q_len
    ([1000, 90, 1], 32, 8, 2, 64, 1, 100, 4),
    ([1000, 350], 64, 5, 1, 128, 2, 33, 70),     # sinks over more than a tile
    ([300], 256, 3, 3, 32, 4, 1, 0),             # a window of the token itself
    ([900], 16, 4, 4, 64, 1, 5000, 10),          # a window longer than the sequence
    ([40000, 7, 9000, 130], 128, 8, 2, 128, 1, 0, 0),  # one long sequence among short ones
]


@pytest.mark.parametrize("lengths,page,heads,kv_heads,head_dim,q_len,window,sinks", ATTENDS)
@pytest.mark.parametrize("dtype", [E4M3, BF16])
@pytest.mark.parametrize("room", [0, 1 << 17])
def test_attend(lengths, page, heads, kv_heads, head_dim, q_len, window, sinks, dtype, room):
    """`room`: tokens that the page table has columns for. Short tables give each head to one CTA, long ones (without a
    window) cut the heads into stretches."""
    cache, seqs = _filled(lengths, page, kv_heads, head_dim, dtype, sum(lengths) + heads)
    seqs.table = torch.nn.functional.pad(seqs.table, (0, max(0, room // page - seqs.table.shape[1])), value=-1)
    g = _gen(heads)
    rows = len(lengths) * q_len
    packed = torch.randn(rows, heads * head_dim + 16, generator=g).bfloat16().cuda()
    q = packed[:, 8:8 + heads * head_dim]
    out = torch.full((rows, heads * head_dim + 8), 5.0, dtype=BF16, device="cuda")[:, :heads * head_dim]
    args = dict(q_len=q_len, window=window, sinks=sinks)
    cache.attend(q, seqs.table.cuda(), _i32(lengths), out=out, **args)
    _check_attend(cache, seqs, lengths, heads, q_len, window, sinks, q, out, head_dim**-0.5)
    again = cache.attend(q, seqs.table.cuda(), _i32(lengths), **args)
    assert torch.equal(out, again)  # the join's order does not depend on who comes last


@pytest.mark.parametrize("dtype", [E4M3, BF16])
def test_attend_scores_far_apart(dtype):
    """Scores of several hundred, growing along the sequence (the running maximum moves), and page scales 2^30 apart."""
    n, d = 600, 64
    seqs = _Sequences([n], 16, 5)
    cache = serving.KVCache.allocate(seqs.pages, 1, d, 16, dtype)
    g = _gen(7)
    qkv = torch.randn(n, 3 * d, generator=g)
    qkv[:, d:2 * d] *= torch.linspace(0.1, 60.0, n)[:, None]
    qkv[:, 2 * d:] *= torch.exp2(torch.arange(n) // 16 % 31 - 15.0)[:, None]
    cache.append(qkv.bfloat16().cuda(), 1, _i32([0]), _i32([n]), _i32([0]), seqs.table.cuda(), n)
    q = (torch.randn(1, 4 * d, generator=g) * torch.tensor([1e-3, 1.0, 10.0, 200.0]).repeat_interleave(d)).bfloat16().cuda()
    out = cache.attend(q, seqs.table.cuda(), _i32([n]))
    _check_attend(cache, seqs, [n], 4, 1, 0, 0, q, out, d**-0.5)


@pytest.mark.parametrize("room", [0, 1 << 17])
def test_attend_many_sequences_and_workspace_reuse(room):
    """More sequences than threads of a CTA, then a smaller and a larger call on the same stream's workspace."""
    lengths = [(37 * b) % 90 for b in range(300)]
    cache, seqs = _filled([max(1, n) for n in lengths], 16, 2, 32, E4M3, 9)
    table = torch.nn.functional.pad(seqs.table, (0, max(0, room // 16 - seqs.table.shape[1])), value=-1).cuda()
    q = torch.randn(300, 4 * 32, generator=_gen(3)).bfloat16().cuda()
    out = cache.attend(q, table, _i32(lengths))
    _check_attend(cache, seqs, lengths, 4, 1, 0, 0, q, out, 32**-0.5)
    one = cache.attend(q[7:8], table[7:8], _i32(lengths[7:8]))
    assert torch.equal(one, out[7:8])
    two = cache.attend(q[:100].reshape(100, 128), table[:50], _i32(lengths[:50]), q_len=2)
    _check_attend(cache, seqs, lengths[:50], 4, 2, 0, 0, q[:100], two, 32**-0.5)
    assert torch.equal(cache.attend(q, table, _i32(lengths)), out)


@pytest.mark.parametrize("head_dim,heads,dtype", [(64, 3, E4M3), (128, 12, E4M3), (128, 4, E4M3), (128, 10, BF16),
                                                  (64, 16, BF16), (32, 1, BF16), (128, 8, BF16)])
@pytest.mark.parametrize("room", [0, 1 << 17])
def test_attend_more_sequences_than_sms(head_dim, heads, dtype, room):
    """A quarter of an SM to each sequence, or stretches that hold several of them."""
    lengths = [(53 * b) % 211 for b in range(160)]
    cache, seqs = _filled([max(1, n) for n in lengths], 32, 1, head_dim, dtype, 3)
    table = torch.nn.functional.pad(seqs.table, (0, max(0, room // 32 - seqs.table.shape[1])), value=-1)
    q = torch.randn(160, heads * head_dim, generator=_gen(3)).bfloat16().cuda()
    out = cache.attend(q, table.cuda(), _i32(lengths))
    _check_attend(cache, seqs, lengths, heads, 1, 0, 0, q, out, head_dim**-0.5)


@pytest.mark.parametrize("batch", [1, 2, 3, 6, 9])  # clusters of 8 for 2 ... 12 heads, of 4 up to 32, of 2 up to 64
@pytest.mark.parametrize("kv_heads,head_dim,heads,q_len,window,sinks,dtype", [
    (2, 128, 8, 1, 0, 0, E4M3), (7, 64, 7, 1, 0, 0, BF16), (6, 128, 18, 3, 0, 0, BF16), (4, 32, 4, 2, 0, 0, E4M3),
    (4, 64, 20, 2, 1500, 20, E4M3), (1, 128, 20, 1, 0, 0, E4M3), (7, 128, 14, 1, 2000, 4, BF16)])
def test_attend_clusters(batch, kv_heads, head_dim, heads, q_len, window, sinks, dtype):
    lengths = [2700, 0, 17, 1301, 640, 1, 2499, 128, 3][:batch]
    cache, seqs = _filled([max(1, n) for n in lengths], 64, kv_heads, head_dim, dtype, batch)
    q = torch.randn(batch * q_len, heads * head_dim, generator=_gen(5)).bfloat16().cuda()
    args = dict(q_len=q_len, window=window, sinks=sinks)
    out = cache.attend(q, seqs.table.cuda(), _i32(lengths), **args)
    _check_attend(cache, seqs, lengths, heads, q_len, window, sinks, q, out, head_dim**-0.5)
    assert torch.equal(cache.attend(q, seqs.table.cuda(), _i32(lengths), **args), out)


@pytest.mark.parametrize("room", [0, 1 << 17])
def test_attend_on_another_stream_and_in_a_graph(room):
    lengths = [3000, 11]
    cache, seqs = _filled(lengths, 32, 2, 64, E4M3, 4)
    table = torch.nn.functional.pad(seqs.table, (0, max(0, room // 32 - seqs.table.shape[1])), value=-1).cuda()
    n = _i32(lengths)
    q = torch.randn(2, 8 * 64, generator=_gen(3)).bfloat16().cuda()
    want = cache.attend(q, table, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cache.attend(q, table, n)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attend(q, table, n, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)


def test_attend_indices_outside_their_tables():
    cache, seqs = _filled([40], 16, 1, 32, E4M3, 1)
    q = torch.randn(1, 32, generator=_gen(1)).bfloat16().cuda()
    table = seqs.table.cuda()
    wide = torch.nn.functional.pad(table, (0, 8192), value=1000)
    for bad_table, n, site in ((table, 49, 1), (table, -1, 1), (torch.full_like(table, 1000), 40, 2), (wide, 60, 2),
                               (wide, 1 << 20, 1), (wide, -1, 1)):
        cache.attend(q, bad_table, _i32([n]))
        torch.cuda.synchronize()
        assert _capi.device_status(clear=True) == (7 << 16) | (site << 8) | 3


def test_cache_slices_of_one_buffer():
    """K and V as halves of one buffer (strides above the dense ones), offsets past 2^31 elements reached by the last page."""
    pages, hk, page, d = 70000, 4, 64, 64
    both = torch.empty(pages, 2, hk, page, d, dtype=E4M3, device="cuda")  # 2.3 G elements
    cache = serving.KVCache(both[:, 0], both[:, 1], torch.ones(pages, hk, device="cuda"),
                            torch.ones(pages, hk, device="cuda"))
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32)
    n = 150
    qkv = torch.randn(n, 3 * hk * d, generator=_gen(6)).bfloat16()
    cache.append(qkv.cuda(), hk, _i32([0]), _i32([n]), _i32([0]), table.cuda(), n)
    q = torch.randn(1, hk * d, generator=_gen(8)).bfloat16().cuda()
    out = cache.attend(q, table.cuda(), _i32([n]))
    ids = table[0].long().cuda()
    small = serving.KVCache(cache.k.view(torch.uint8)[ids].view(E4M3), cache.v.view(torch.uint8)[ids].view(E4M3),
                            cache.k_scale[ids], cache.v_scale[ids])
    seqs = _Sequences([n], page, 0)
    seqs.table = torch.tensor([[0, 1, 2]], dtype=torch.int32)
    _check_attend(small, seqs, [n], hk, 1, 0, 0, q, out, d**-0.5)
    v = _gather(small, "v", seqs.table[0], n)
    exact = qkv.double().view(n, 3, hk, d)[:, 2].transpose(0, 1)
    _close(v, exact, 2**-4 * exact.abs() + 2**-9)


# ---------------------------------------------------------------------------------- prompt attention with a window
WINDOWS = [
    # batch, seq, heads, kv_heads, head_dim, window, sinks
    (1, 1, 1, 1, 64, 0, 0),
    (2, 77, 4, 4, 64, 32, 4),
    (1, 300, 4, 1, 128, 100, 20),
    (2, 129, 3, 3, 32, 1, 0),
    (1, 517, 6, 2, 64, 130, 1),       # a group of three: no packing
    (1, 400, 12, 2, 128, 64, 0),      # a group of six: two heads to a tile
    (1, 1000, 16, 1, 64, 256, 130),   # sixteen heads to a tile; sinks over more than a tile
    (1, 260, 32, 1, 32, 40, 16),      # thirty-two heads: two tiles of sixteen
    (3, 640, 2, 2, 128, 128, 0),
    (1, 1100, 8, 4, 64, 0, 0),
    (2, 700, 2, 1, 128, 699, 3),
    (1, 900, 1, 1, 128, 300, 600),    # sinks beyond the window
]


def _check_window(q, k, v, out, batch, seq, heads, kv_heads, d, window, sinks, lengths, scale):
    q, k, v = (x.cpu().double().view(batch, seq, -1, d) for x in (q, k, v))
    got = out.cpu().view(batch, seq, heads, d)
    for b in range(batch):
        n = lengths[b]
        assert not bool(got[b, n:].any())
        seen = oracle.visible_keys(torch.arange(n), n, window, sinks)
        for h in range(heads):
            ref, absum, size = oracle.attend(q[b, :n, h], k[b, :n, h * kv_heads // heads], v[b, :n, h * kv_heads // heads],
                                             seen, scale)
            _close(got[b, :n, h], ref, 2**-8 * ref.abs() + (2**-8 + 2**-12 + 2 * d * 2**-23 * size) * absum)


@pytest.mark.parametrize("batch,seq,heads,kv_heads,d,window,sinks", WINDOWS)
@pytest.mark.parametrize("ragged", [False, True])
def test_window_attention(batch, seq, heads, kv_heads, d, window, sinks, ragged):
    g = _gen(seq + heads)
    width = (heads + 2 * kv_heads) * d
    packed = torch.randn(batch * seq, width + 8, generator=g).bfloat16()
    lengths = [seq] * batch
    if ragged:
        lengths = [max(0, seq - 1 - 61 * b) for b in range(batch)]
        for b, n in enumerate(lengths):
            packed[b * seq + n:(b + 1) * seq] = math.nan  # what padding rows hold
    packed = packed.cuda()
    q, k, v = packed[:, :heads * d], packed[:, heads * d:(heads + kv_heads) * d], packed[:, (heads + kv_heads) * d:width]
    out = torch.full((batch * seq, heads * d + 16), 3.0, dtype=BF16, device="cuda")[:, 8:8 + heads * d]
    serving.window_attention(q, k, v, batch, seq, d, window=window, sinks=sinks,
                             kv_len=_i32(lengths) if ragged else None, out=out)
    _check_window(q, k, v, out, batch, seq, heads, kv_heads, d, window, sinks, lengths, d**-0.5)


@pytest.mark.parametrize("d", [64, 128])
def test_window_attention_scores_far_apart(d):
    """The running maximum moves by far more than the rescale threshold, up and down along the list."""
    n = 700
    g = _gen(d)
    q, k, v = (torch.randn(n, 2 * d, generator=g) for _ in range(3))
    k *= torch.linspace(0.1, 40.0, n)[:, None] * torch.where(torch.arange(n) % 300 < 150, 1.0, 0.01)[:, None]
    q, k, v = (x.bfloat16().cuda() for x in (q, k, v))
    for window, sinks in ((0, 0), (200, 5)):
        out = serving.window_attention(q, k, v, 1, n, d, window=window, sinks=sinks)
        _check_window(q, k, v, out, 1, n, 2, 2, d, window, sinks, [n], d**-0.5)


@pytest.mark.parametrize("d", [32, 64, 128])
def test_window_attention_without_a_window_is_causal_attention(d):
    batch, seq, heads = 2, 333, 2
    qkv = torch.randn(batch * seq, 3 * heads * d, generator=_gen(d)).bfloat16().cuda()
    ctx = torch.empty(batch * seq, heads * d, dtype=BF16, device="cuda")
    _capi.attention(qkv, batch, seq, heads, d, 0, heads * d, 2 * heads * d, None, True, d**-0.5, ctx)
    parts = qkv.split(heads * d, 1)
    for window in (0, seq, 1 << 40):
        out = serving.window_attention(*parts, batch, seq, d, window=window)
        assert float((out.float() - ctx.float()).abs().max()) <= 2**-6 * float(ctx.float().abs().max())


def test_window_attention_long_sequence_tail():
    """Far positions (the head-major order, list places of a long band): the last rows of 20000 against 64 bits."""
    n, d, window, sinks = 20000, 64, 3000, 7
    qkv = torch.randn(n, 6 * d, generator=_gen(2)).bfloat16().cuda()
    q, k, v = qkv[:, :4 * d], qkv[:, 4 * d:5 * d], qkv[:, 5 * d:]
    out = serving.window_attention(q, k, v, 1, n, d, window=window, sinks=sinks)
    rows = torch.tensor([0, 31, 3000, 3007, 9999, 19968, 19999])
    seen = oracle.visible_keys(rows, n, window, sinks)
    for h in range(4):
        ref, absum, size = oracle.attend(q.cpu().double().view(n, 4, d)[rows, h], k.cpu().double(), v.cpu().double(), seen,
                                         d**-0.5)
        _close(out.view(n, 4, d)[rows.cuda(), h], ref, 2**-8 * ref.abs() + (2**-8 + 2**-12 + 2 * d * 2**-23 * size) * absum)


# ---------------------------------------------------------------------------------- refusals of the wrappers
def test_wrappers_refuse_what_does_not_fit():
    table = serving.rotary_table(16, 32)
    x = torch.zeros(4, 64, dtype=BF16, device="cuda")
    pos = _i32([0, 1, 2, 3])
    for bad in (dict(x=x.float()), dict(x=x.t()), dict(x=x[:, :40]), dict(positions=pos[:3]), dict(positions=pos.long()),
                dict(table=table.double()), dict(table=table[:, :, :1]), dict(out=x[:3]), dict(x=x.view(2, 2, 64))):
        with pytest.raises((ValueError, IndexError)):
            serving.rotary(**(dict(x=x, positions=pos, table=table, head_dim=32, out=torch.empty_like(x)) | bad))
    cache = serving.KVCache.allocate(4, 2, 32, 16)
    qkv = torch.zeros(4, 8 * 32, dtype=BF16, device="cuda")
    pages = _i32([[0, 1], [2, 3]])
    good = dict(qkv=qkv, num_heads=4, new_start=_i32([0, 2]), new_len=_i32([2, 2]), past_len=_i32([0, 0]),
                page_table=pages, max_new=2)
    for bad in (dict(num_heads=2), dict(new_start=_i32([0])), dict(page_table=pages[:1]), dict(page_table=pages.repeat(1, 2)[:, ::2]),
                dict(past_len=torch.zeros(2, device="cuda")), dict(q_out=qkv[:, :128]), dict(table=table, q_out=qkv[:, :96]),
                dict(k_out=qkv[:2, :64])):
        with pytest.raises((ValueError, RuntimeError)):
            cache.append(**(good | bad))
    q = torch.zeros(2, 4 * 32, dtype=BF16, device="cuda")
    good = dict(q=q, page_table=pages, kv_len=_i32([1, 1]))
    for bad in (dict(q_len=2), dict(q=q[:, :48]), dict(q=q[:, :96]), dict(kv_len=_i32([1])), dict(sinks=2), dict(scale=0.0),
                dict(workspace=torch.zeros(256, dtype=torch.uint8, device="cuda")),
                dict(workspace=torch.zeros(1 << 20, device="cuda")), dict(out=q[:, :64])):
        with pytest.raises((ValueError, RuntimeError)):
            cache.attend(**(good | bad))
    for bad in ((q, q[:, :64], q, 1, 2), (q, q, q, 2, 2), (q, q[:, :40], q[:, :40], 1, 2)):
        with pytest.raises(ValueError):
            serving.window_attention(*bad, 32)
    with pytest.raises(RuntimeError, match="sinks"):
        serving.window_attention(q, q, q, 1, 2, 32, sinks=1)
    k = torch.zeros(4, 2, 16, 32, dtype=BF16, device="cuda")
    for bad in ((k, k[:2]), (k, k.float()), (k.half(), k.half()), (k[:, :, :8], k[:, :, :8]),
                (k, k, torch.ones(4, 2, device="cuda"), torch.ones(4, 2, device="cuda")), (k.to(E4M3), k.to(E4M3)),
                (k.transpose(2, 3), k.transpose(2, 3))):
        with pytest.raises(ValueError):
            serving.KVCache(*bad)
