"""The 4-bit cache and reading a cache back, on a B200, against 64-bit restatements.

A code is made by operations that are exact for bf16 values (or rounded one by one), so what is stored of values that
were not turned is compared bit for bit. Turned keys differ from 64 bits by some 2^-24 of their size: a code, a step or a
middle at a border may then be its neighbour. Any stored value is within 0.55 steps and 2^-8 of its middle of the
value given: half a step, 8 * 2^-9 of one for the factor's rounding, 15 * 2^-9 of one for the step's at the ends, and
the middle's own rounding.

Attention: with steps s and middles m of a token's groups, a weight is rounded to fp16 (2^-11 of itself), its product with a
step again, and a step or a middle loses at most 2^-25 of a power of two up to twice the largest parameter; the output is bf16. A
score's fp32 sums begin at -1032 sum(q) (72 for half of the elements) and add q (1024 + code): 34 terms of at most 2071 |q|, off by
2^-23 each in the worst case. A middle meets the sum of q over its group in two bf16 terms: the first is off by half a step, 2^-8
of the sum's power of two, the second by 2^-8 of that one's, 2^-9 at most: 2^-17, or 64 * 2^-23, of sum |q| besides the 20
fp32 sums. That worst case is far from what happens (the terms' errors are not alike),
so the whole output is also held to 2^-8 of its norm, twice what its own rounding may take.
"""

import math

import pytest
import torch

from oracle import serving_fp64 as oracle
from tiktoktechjam2026track3_b200 import _capi, serving

pytestmark = pytest.mark.gpu

BF16, E4M3, INT4 = torch.bfloat16, torch.float8_e4m3fn, torch.uint8


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


def _starts(lengths):
    return [sum(lengths[:b]) for b in range(len(lengths))]


def _close(got, ref, bound):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    off = (got - ref).abs() - bound
    assert not bool((off > 0).any()), f"{float(off.nan_to_num().max())} above the bound"


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


def _decode(cache, which):
    """Every value of the cache, float64 [pages, kv_heads, page_size, head_dim]."""
    x, scale = (cache.k, cache.k_scale) if which == "k" else (cache.v, cache.v_scale)
    if cache.k.dtype == INT4:
        return oracle.int4_decode(x.cpu(), scale.cpu())
    y = x.cpu().double() if scale is None else x.cpu().float().double()
    return y if scale is None else y * scale.cpu().double()[:, :, None, None]


def _of(values, table, page, first, last):
    """Tokens first ... last - 1 of a sequence, [heads, tokens, head_dim]."""
    if first >= last:
        return values[0][:, :0]
    ids = table[first // page:-(-last // page)].long()
    x = values[ids].transpose(0, 1).flatten(1, 2)
    return x[:, first % page:first % page + last - first]


def _junk(cache):
    """Random codes and NaN parameters (or values) in every slot."""
    g = _gen(99)
    for x, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        if cache.k.dtype == INT4:
            x.copy_(torch.randint(0, 256, x.shape, generator=g, dtype=torch.uint8))
            scale.fill_(math.nan)
        else:
            x.copy_(torch.full(x.shape, math.nan).to(x.dtype))


# ---------------------------------------------------------------------------------- append
APPENDS = [
    # new, past, page_size, heads, kv_heads, head_dim, rotary_dim, interleaved
    ([1], [0], 16, 1, 1, 32, 32, False),
    ([1, 1, 1], [15, 16, 0], 16, 4, 2, 64, 64, False),
    ([5, 0, 40], [31, 7, 33], 32, 3, 3, 64, 32, True),
    ([130, 1], [0, 200], 64, 10, 2, 128, 128, False),
    ([77, 300, 3], [60, 1, 127], 128, 6, 1, 128, 48, True),
    ([17], [250], 256, 2, 2, 256, 256, False),
    ([33, 4], [3, 40], 32, 4, 2, 96, 80, False),  # an odd number of groups, pairs across groups
    ([19], [5], 16, 1, 1, 160, 16, True),
    ([21, 2], [0, 9], 16, 9, 3, 32, 16, False),
]


@pytest.mark.parametrize("new,past,page,heads,kv_heads,head_dim,rotary_dim,interleaved", APPENDS)
@pytest.mark.parametrize("rotated", [True, False])
def test_append(new, past, page, heads, kv_heads, head_dim, rotary_dim, interleaved, rotated):
    g = _gen(sum(new) + page)
    seqs = _Sequences([n + p for n, p in zip(new, past)], page, 3)
    cache = serving.KVCache.allocate(seqs.pages, kv_heads, head_dim, page, INT4)
    _junk(cache)
    table = serving.rotary_table(2048, rotary_dim) if rotated else None
    step = dict(table=table, interleaved=interleaved)
    pages = seqs.table.cuda()

    def rows(n):
        x = torch.randn(n, (heads + 2 * kv_heads) * head_dim, generator=g) * torch.exp2(torch.randint(-6, 7, (n, 1), generator=g))
        x[:, ::29] *= 6
        return x.bfloat16()

    first = rows(sum(past))
    if sum(past):
        cache.append(first.cuda(), heads, _i32(_starts(past)), _i32(past), _i32([0] * len(past)), pages, max(past), **step)
    before = [x.clone() for x in (cache.k, cache.k_scale, cache.v, cache.v_scale)]
    qkv = rows(sum(new))
    k_out = torch.full((sum(new), kv_heads * head_dim), 9.0, dtype=BF16, device="cuda")
    q_out = cache.append(qkv.cuda(), heads, _i32(_starts(new)), _i32(new), _i32(past), pages, max(new), k_out=k_out, **step)
    x = qkv.double().view(-1, heads + 2 * kv_heads, head_dim)
    keys = x[:, heads:heads + kv_heads]
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
        assert torch.equal(k_out.cpu().double().view(-1, kv_heads, head_dim), keys)
    slots = [(int(seqs.table[b, (p + i) // page]), (p + i) % page) for b, (n, p) in enumerate(zip(new, past)) for i in range(n)]
    for which, fresh in (("k", keys), ("v", x[:, heads + kv_heads:])):
        now = _decode(cache, which)
        got = torch.stack([now[page_id, :, slot] for page_id, slot in slots])
        if which == "k" and rotated:
            s, m = (z.repeat_interleave(32, -1) for z in oracle.int4_params(fresh))
            assert int((got != oracle.int4(fresh)).sum()) <= 32 + got.numel() // 2000
            _close(got, fresh, 0.55 * 1.01 * s + 2**-8 * 1.01 * m.abs() + 2**-21 * fresh.abs().amax(-1, keepdim=True))
        else:
            assert torch.equal(got, oracle.int4(fresh))
    # Everything else, earlier tokens among it, is as it was.
    for x, was in zip((cache.k, cache.k_scale, cache.v, cache.v_scale), before):
        x, was = x.cpu().view(torch.uint8), was.cpu().view(torch.uint8)
        for page_id, slot in slots:
            was[page_id, :, slot] = x[page_id, :, slot]
        assert torch.equal(x, was)


def test_tokens_one_by_one_or_together_are_the_same_codes():
    heads, kv_heads, d, n = 4, 2, 64, 45
    seqs = _Sequences([n], 16, 1)
    table, pages = serving.rotary_table(128, 48), seqs.table.cuda()
    qkv = torch.randn(n, (heads + 2 * kv_heads) * d, generator=_gen(2)).bfloat16().cuda()
    caches = [serving.KVCache.allocate(seqs.pages, kv_heads, d, 16, INT4) for _ in range(2)]
    q = caches[0].append(qkv, heads, _i32([0]), _i32([n]), _i32([0]), pages, n, table=table)
    for i in range(n):
        one = caches[1].append(qkv, heads, _i32([i]), _i32([1]), _i32([i]), pages, 1, table=table)
        assert torch.equal(one[i], q[i])
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(caches[0], name), getattr(caches[1], name))


@pytest.mark.parametrize("d,rotary_dim", [(64, 64), (96, 96), (128, 32)])
def test_append_in_place_matches_separate_outputs(d, rotary_dim):
    heads, kv_heads = 6, 2
    seqs = _Sequences([70], 32, 1)
    table = serving.rotary_table(128, rotary_dim)
    qkv = torch.randn(70, (heads + 2 * kv_heads) * d, generator=_gen(2)).bfloat16().cuda()
    got = []
    for in_place in (False, True):
        cache = serving.KVCache.allocate(seqs.pages, kv_heads, d, 32, INT4)
        x = qkv.clone()
        q = x[:, :heads * d] if in_place else torch.empty(70, heads * d, dtype=BF16, device="cuda")
        k = x[:, heads * d:(heads + kv_heads) * d] if in_place else torch.empty(70, kv_heads * d, dtype=BF16, device="cuda")
        cache.append(x, heads, _i32([0]), _i32([70]), _i32([0]), seqs.table.cuda(), 70, table=table, q_out=q, k_out=k)
        got.append((q.clone(), k.clone(), cache.k, cache.v, cache.k_scale, cache.v_scale))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_append_odd_groups():
    """Values halfway between codes, groups of one value, tiny and huge ranges, values that are not finite."""
    d = 32
    rows = torch.zeros(9, d)
    rows[0] = torch.arange(d) % 16                        # least 0, step 1
    rows[0, 3:8] = torch.tensor([0.5, 1.5, 2.5, 6.5, 14.5])
    rows[1] = 3.0                                         # no range: the middle alone
    rows[2] = 100.0
    rows[2, 5] = 100.5                                    # a range below the middle's rounding
    rows[3] = 0.0
    rows[3, 1] = 2.0**-105                                # a step below 2^-100
    rows[4], rows[4, 0] = 1.0, math.nan
    rows[5], rows[5, 31] = 1.0, math.inf
    rows[6], rows[6, 7], rows[6, 8] = 1.0, math.inf, -math.inf
    rows[7] = torch.linspace(-2.0**120, 2.0**120, d)
    rows[8] = torch.linspace(-1.0, 1.0, d) * 2.0**-90
    qkv = torch.cat([torch.zeros(9, d), rows, rows.flip(1)], 1).bfloat16()
    cache = serving.KVCache.allocate(1, 1, d, 16, INT4)
    cache.append(qkv.cuda(), 1, _i32([0]), _i32([9]), _i32([0]), _i32([[0]]), 9)
    given = qkv.double()
    for which, x in (("k", given[:, d:2 * d]), ("v", given[:, 2 * d:])):
        got, ref = _decode(cache, which)[0, 0, :9], oracle.int4(x)
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        assert torch.equal(got.nan_to_num(), ref.nan_to_num())
    assert bool(torch.isnan(_decode(cache, "k")[0, 0, 4:7]).all())
    assert _decode(cache, "k")[0, 0, 0, 3:8].tolist() == [0.0, 2.0, 2.0, 6.0, 14.0]


def test_append_indices_outside_their_tables_write_nothing():
    qkv = torch.ones(4, 96, dtype=BF16, device="cuda")
    for start, count, past, pages in ((0, 5, 0, [[0, 1]]), (2, 3, 0, [[0, 1]]), (0, 4, 30, [[0, 1]]), (0, 4, 0, [[9, 1]]),
                                      (-1, 2, 0, [[0, 1]]), (0, 4, -2, [[0, 1]]), (0, 3, 0, [[-1, -1]])):
        cache = serving.KVCache.allocate(2, 1, 32, 16, INT4)
        cache.append(qkv, 1, _i32([start]), _i32([count]), _i32([past]), _i32(pages), 4)
        torch.cuda.synchronize()
        status = _capi.device_status(clear=True)
        assert status >> 16 == 6 and status & 0xFF == 3
        assert not bool(cache.k.any()) and not bool(cache.k_scale.any())


# ---------------------------------------------------------------------------------- reading back
def _filled(lengths, page, kv_heads, d, dtype, seed):
    """A cache with random keys and values, junk in every slot that no sequence uses."""
    seqs = _Sequences(lengths, page, seed)
    g = _gen(seed)
    cache = serving.KVCache.allocate(seqs.pages, kv_heads, d, page, dtype)
    _junk(cache)
    n = sum(lengths)
    qkv = torch.randn(n, 3 * kv_heads * d, generator=g)
    qkv[:, ::29] *= 5
    qkv *= torch.exp2(torch.randint(-2, 3, (n, 1), generator=g))
    cache.append(qkv.bfloat16().cuda(), kv_heads, _i32(_starts(lengths)), _i32(lengths), _i32([0] * len(lengths)),
                 seqs.table.cuda(), max(lengths))
    return cache, seqs


READS = [
    # lengths, start, take, page_size, kv_heads, head_dim
    ([1], [0], [1], 16, 1, 32),
    ([40, 17, 3], [0, 16, 1], [40, 1, 2], 16, 3, 64),
    ([130, 1, 257], [33, 0, 200], [60, 0, 57], 64, 2, 128),
    ([77, 5], [70, 5], [7, 0], 32, 4, 96),
    ([300], [1], [299], 256, 1, 256),
    ([9, 700], [2, 0], [3, 700], 128, 5, 32),
]


@pytest.mark.parametrize("lengths,start,take,page,kv_heads,d", READS)
@pytest.mark.parametrize("dtype", [INT4, E4M3, BF16])
def test_read(lengths, start, take, page, kv_heads, d, dtype):
    cache, seqs = _filled(lengths, page, kv_heads, d, dtype, 7)
    gaps = [sum(take[:b]) + 2 * b + 1 for b in range(len(take))]  # rows between the sequences belong to nobody
    rows = gaps[-1] + take[-1] + 3
    k_out = torch.full((rows, kv_heads * d + 8), 7.0, dtype=BF16, device="cuda")
    v_out = torch.full((rows, kv_heads * d), 7.0, dtype=BF16, device="cuda")
    got = cache.read(_i32(gaps), _i32(take), _i32(start), seqs.table.cuda(), max(take), k_out=k_out[:, :kv_heads * d],
                     v_out=v_out)
    assert got[1] is v_out
    for which, out in (("k", k_out), ("v", v_out)):
        expect = torch.full(out.shape, 7.0).bfloat16()
        values = _decode(cache, which)
        for b, (first, n) in enumerate(zip(start, take)):
            x = _of(values, seqs.table[b], page, first, first + n)
            expect[gaps[b]:gaps[b] + n, :kv_heads * d] = x.transpose(0, 1).flatten(1).float().bfloat16()
        assert torch.equal(out.cpu(), expect)
        alone = torch.full_like(out, 7.0)
        args = {f"{which}_out": alone[:, :kv_heads * d]}
        cache.read(_i32(gaps), _i32(take), _i32(start), seqs.table.cuda(), max(take), **args)
        assert torch.equal(alone, out)


@pytest.mark.parametrize("d", [16, 48, 240])
@pytest.mark.parametrize("dtype", [E4M3, BF16])
def test_read_other_head_dims(d, dtype):
    cache, seqs = _filled([50, 3], 32, 2, d, dtype, 3)
    k, v = (torch.zeros(53, 2 * d, dtype=BF16, device="cuda") for _ in range(2))
    cache.read(_i32([0, 50]), _i32([50, 3]), _i32([0, 0]), seqs.table.cuda(), 50, k_out=k, v_out=v)
    for which, out in (("k", k), ("v", v)):
        values = _decode(cache, which)
        expect = torch.cat([_of(values, seqs.table[b], 32, 0, n).transpose(0, 1).flatten(1) for b, n in enumerate([50, 3])])
        assert torch.equal(out.cpu(), expect.float().bfloat16())


@pytest.mark.parametrize("dtype", [INT4, E4M3, BF16])
def test_read_indices_outside_their_tables_write_nothing(dtype):
    cache, _ = _filled([40], 16, 1, 32, dtype, 1)
    for out_start, length, start, pages in ((0, 9, 0, [[0, 1]]), (5, 4, 0, [[0, 1]]), (-1, 2, 0, [[0, 1]]), (0, 4, -1, [[0, 1]]),
                                            (0, 4, 29, [[0, 1]]), (0, 4, 0, [[99, 1]]), (0, 4, 0, [[-1, -1]])):
        k, v = (torch.full((8, 32), 7.0, dtype=BF16, device="cuda") for _ in range(2))
        cache.read(_i32([out_start]), _i32([length]), _i32([start]), _i32(pages), 8, k_out=k, v_out=v)
        torch.cuda.synchronize()
        status = _capi.device_status(clear=True)
        assert status >> 16 == 8 and status & 0xFF == 3
        assert bool((k == 7.0).all()) and bool((v == 7.0).all())


# ---------------------------------------------------------------------------------- attention
def _check_attend(cache, seqs, lengths, heads, q_len, window, sinks, q, out, scale):
    d, hk, page = cache.head_dim, cache.kv_heads, cache.page_size
    q64 = q.cpu().double().view(len(lengths), q_len, heads, d)
    got = out.cpu().view(len(lengths), q_len, heads, d)
    k_all, v_all = _decode(cache, "k"), _decode(cache, "v")
    params = {w: getattr(cache, w + "_scale").cpu().double() for w in "kv"}

    def of(values, b, n):
        return _of(values, seqs.table[b], page, 0, n)

    for b, n in enumerate(lengths):
        k, v = of(k_all, b, n), of(v_all, b, n)
        ks, km = (of(params["k"][..., i, :], b, n).abs() for i in (0, 1))
        vm = of(params["v"][..., 1, :], b, n).repeat_interleave(32, -1)
        seen = oracle.visible_keys(torch.arange(n - q_len, n), n, window, sinks)
        used = seen.any(0)
        for h in range(heads):
            g = h * hk // heads
            x = q64[b, :, h]
            ref, absum, _ = oracle.attend(x, k[g], v[g], seen, scale)
            mid_ref, mid_sum, _ = oracle.attend(x, k[g], vm[g], seen, scale)
            part_sum = oracle.attend(x, k[g], v[g] - vm[g], seen, scale)[1]
            share = x.abs().view(q_len, d // 32, 32).sum(-1)
            off = scale * 2**-23 * (34 * 2071 * share @ ks[g].T + (20 + 64) * share @ km[g].T)
            off = torch.where(used, off, 0.0).amax(-1, keepdim=True) if n else torch.zeros(q_len, 1, dtype=torch.float64)
            _close(got[b, :, h], ref, 2**-8 * ref.abs() + 2**-10 * part_sum + 2**-11 * mid_sum + (2.1 * off + 2**-18) * absum
                   + 2**-20 * params["v"][seqs.table[b, :-(-n // page)].long()].nan_to_num().abs().max() if n else 0 * ref)
            assert float((got[b, :, h].double() - ref).norm()) <= 2**-8 * float(ref.norm()) + 2**-18


ATTENDS = [
    # lengths, page_size, heads, kv_heads, head_dim, q_len, window, sinks
    ([1], 16, 1, 1, 64, 1, 0, 0),
    ([0, 5, 16, 17], 16, 2, 1, 32, 1, 0, 0),
    ([100, 1000, 31], 16, 12, 12, 64, 1, 0, 0),
    ([257, 64], 64, 10, 2, 128, 1, 0, 0),
    ([2000], 128, 16, 1, 128, 1, 0, 0),          # 16 query heads of one key head: one block of 16 rows
    ([700, 3], 32, 20, 1, 64, 1, 0, 0),          # 20: two blocks
    ([500, 130, 2], 16, 6, 2, 128, 3, 0, 0),     # drafts; a sequence shorter than q_len
    ([333, 8], 16, 12, 1, 32, 2, 0, 0),
    ([1000, 90, 1], 32, 8, 2, 64, 1, 100, 4),
    ([1000, 350], 64, 5, 1, 128, 2, 33, 70),     # sinks over more than a tile
    ([300], 256, 3, 3, 32, 4, 1, 0),             # a window of the token itself
    ([900], 16, 4, 4, 64, 1, 5000, 10),          # a window longer than the sequence
    ([20000, 7, 5000, 130], 128, 8, 2, 128, 1, 0, 0),  # one long sequence among short ones
]


@pytest.mark.parametrize("lengths,page,heads,kv_heads,head_dim,q_len,window,sinks", ATTENDS)
@pytest.mark.parametrize("room", [0, 1 << 17])
def test_attend(lengths, page, heads, kv_heads, head_dim, q_len, window, sinks, room):
    """`room`: tokens that the page table has columns for. Short tables give each head to one CTA, long ones (without a
    window) cut the heads into stretches."""
    cache, seqs = _filled(lengths, page, kv_heads, head_dim, INT4, sum(lengths) + heads)
    seqs.table = torch.nn.functional.pad(seqs.table, (0, max(0, room // page - seqs.table.shape[1])), value=-1)
    rows = len(lengths) * q_len
    packed = torch.randn(rows, heads * head_dim + 16, generator=_gen(heads)).bfloat16().cuda()
    q = packed[:, 8:8 + heads * head_dim]
    out = torch.full((rows, heads * head_dim + 8), 5.0, dtype=BF16, device="cuda")[:, :heads * head_dim]
    args = dict(q_len=q_len, window=window, sinks=sinks)
    cache.attend(q, seqs.table.cuda(), _i32(lengths), out=out, **args)
    _check_attend(cache, seqs, lengths, heads, q_len, window, sinks, q, out, head_dim**-0.5)
    again = cache.attend(q, seqs.table.cuda(), _i32(lengths), **args)
    assert torch.equal(out, again)  # the join's order does not depend on who comes last


@pytest.mark.parametrize("d,heads,kv_heads", [(32, 2, 1), (64, 4, 4), (128, 8, 1)])
@pytest.mark.parametrize("room", [0, 1 << 17])
def test_attend_scores_far_apart(d, heads, kv_heads, room):
    """Queries ten times as large, and of unlike sizes: the maximum moves far, and the weights rest on few tokens."""
    lengths, page = [700, 90], 32
    cache, seqs = _filled(lengths, page, kv_heads, d, INT4, 3)
    seqs.table = torch.nn.functional.pad(seqs.table, (0, max(0, room // page - seqs.table.shape[1])), value=-1)
    q = (torch.randn(2, heads * d, generator=_gen(d)) * 10.0 ** torch.tensor([[1.0], [-3.0]])).bfloat16().cuda()
    out = cache.attend(q, seqs.table.cuda(), _i32(lengths))
    _check_attend(cache, seqs, lengths, heads, 1, 0, 0, q, out, d**-0.5)


@pytest.mark.parametrize("room", [0, 1 << 17])
def test_attend_parameters_far_apart(room):
    """Tokens whose values are 2^12 times those of others, at the start, in the middle and at the end."""
    n, d, page = 600, 64, 16
    seqs = _Sequences([n], page, 1)
    cache = serving.KVCache.allocate(seqs.pages, 1, d, page, INT4)
    _junk(cache)
    qkv = torch.randn(n, 3 * d, generator=_gen(4))
    qkv[:, 2 * d:] *= torch.where(torch.arange(n) % 250 < 3, 2.0**12, 1.0)[:, None]
    cache.append(qkv.bfloat16().cuda(), 1, _i32([0]), _i32([n]), _i32([0]), seqs.table.cuda(), n)
    seqs.table = torch.nn.functional.pad(seqs.table, (0, max(0, room // page - seqs.table.shape[1])), value=-1)
    q = torch.randn(1, d, generator=_gen(5)).bfloat16().cuda()
    out = cache.attend(q, seqs.table.cuda(), _i32([n]))
    _check_attend(cache, seqs, [n], 1, 1, 0, 0, q, out, d**-0.5)
