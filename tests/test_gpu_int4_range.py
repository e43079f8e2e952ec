"""Attention over a 4-bit cache whose values lie far apart, on a B200, against 64-bit restatements.

A token's steps and middles count in a power of two 2^e above them all (e from -60 to 100), and its weight w carries that power, so
that what a token loses is measured by its own w 2^e. Steps are held as fp16 numbers of at most 2^6, middles of at most 2^15: a
subnormal one is off by 2^-25 at most, which is 2^-31 and 2^-40 of 2^e; the weights' largest are 2^7 or more, so that a subnormal
weight, or its product with a step, is off by at most 2^-32 of the largest w 2^e. A code is a whole number of up to 8 steps. Besides
these, a weight is rounded to 2^-11 of itself and its product with a step again; a score's error is that of test_gpu_int4.py, and its
sum with e, of up to 2^8 here, is off by 2^-17 at most, which moves a weight by 2^-17.5 and twice (weight and sum): 2^-16. The output
is bf16.
"""

import math

import pytest
import torch

from test_gpu_int4 import BF16, INT4, _decode, _gen, _i32, _of, _Sequences
from oracle import serving_fp64 as oracle
from tiktoktechjam2026track3_b200 import _capi, serving

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_status(cuda_device):
    _capi.device_status(clear=True)
    yield
    torch.cuda.synchronize()
    assert _capi.device_status(clear=True) == 0


def _cache(k, v, page):
    """A cache of one sequence that holds k and v [tokens, kv_heads, d], rounded to 4 bits."""
    n, kv_heads, d = k.shape
    seqs = _Sequences([n], page, 5)
    cache = serving.KVCache.allocate(seqs.pages, kv_heads, d, page, INT4)
    qkv = torch.cat([torch.zeros(n, kv_heads * d), k.flatten(1), v.flatten(1)], 1).bfloat16().cuda()
    cache.append(qkv, kv_heads, _i32([0]), _i32([n]), _i32([0]), seqs.table.cuda(), n)
    return cache, seqs


def _check(cache, seqs, n, q, out, heads, q_len, window=0, sinks=0, groups=(), table=None):
    """Every element within the bound; the norm of every head's rows, and of those of `groups` by themselves, to 2^-8."""
    d, hk, page, scale = cache.head_dim, cache.kv_heads, cache.page_size, cache.head_dim**-0.5
    k_all, v_all = (_of(_decode(cache, w), seqs.table[0], page, 0, n) for w in "kv")
    k_step, k_mid, v_step, v_mid = (
        _of(getattr(cache, w + "_scale").cpu().double()[..., i, :], seqs.table[0], page, 0, n).abs() for w in "kv" for i in (0, 1))
    seen = oracle.visible_keys(torch.arange(n - q_len, n), n, window, sinks)
    q64, got = q.cpu().double().view(q_len, heads, d), out.cpu().double().view(q_len, heads, d)
    for h in range(heads):
        g, x = h * hk // heads, q64[:, h]
        ref, absum, _ = oracle.attend(x, k_all[g], v_all[g], seen, scale)
        mid_sum = oracle.attend(x, k_all[g], v_mid[g].repeat_interleave(32, -1), seen, scale)[0]
        part_sum = oracle.attend(x, k_all[g], v_all[g] - oracle_middles(cache, seqs, n, g), seen, scale)[1]
        top = torch.maximum(v_step[g], v_mid[g]).amax(-1)
        power = torch.exp2(torch.frexp(top)[1].double().clamp(min=-60))
        weights = oracle.attend(x, k_all[g], torch.eye(n, dtype=torch.float64), seen, scale)[0]
        own, largest = weights @ power[:, None], (weights * power).amax(-1, keepdim=True)
        share = x.abs().view(q_len, d // 32, 32).sum(-1)
        off = scale * 2**-23 * (34 * 2071 * share @ k_step[g].T + (20 + 64) * share @ k_mid[g].T)
        off = torch.where(seen.any(0), off, 0.0).amax(-1, keepdim=True)
        bound = (2**-8 * ref.abs() + 2**-10 * part_sum + 2**-11 * mid_sum + (2.1 * off + 2**-16) * absum
                 + (8 * 2**-31 + 2**-40) * own + n * (1 + 8) * 2**-32 * largest)
        assert bool(torch.isfinite(got[:, h]).all())
        over = (got[:, h] - ref).abs() - bound
        assert not bool((over > 0).any()), f"{float(over.max())} above the bound"
        for part in [slice(0, d)] + [slice(32 * y, 32 * y + 32) for y in groups]:
            assert float((got[:, h, part] - ref[:, part]).norm()) <= 2**-8 * float(ref[:, part].norm())


def oracle_middles(cache, seqs, n, head):
    mid = _of(cache.v_scale.cpu().double()[..., 1, :], seqs.table[0], cache.page_size, 0, n)[head]
    return mid.repeat_interleave(32, -1)


def _attend(cache, seqs, n, q, room, **args):
    table = torch.nn.functional.pad(seqs.table, (0, max(0, room // cache.page_size - seqs.table.shape[1])), value=-1)
    return cache.attend(q, table.cuda(), _i32([n]), **args)


SHAPES = [  # head_dim, heads, kv_heads, q_len, page_size
    (32, 2, 2, 1, 16), (64, 4, 1, 1, 32), (128, 8, 2, 1, 64), (64, 12, 1, 1, 16), (128, 5, 1, 2, 128), (32, 9, 1, 2, 16)]


@pytest.mark.parametrize("d,heads,kv_heads,q_len,page", SHAPES)
@pytest.mark.parametrize("far", [8, 16, 20, 24, 32, 44])
@pytest.mark.parametrize("room", [0, 1 << 17])
def test_large_tokens_of_no_weight(d, heads, kv_heads, q_len, page, far, room):
    """Tokens whose values are 2^far times the others' and whose weight is some 2^-70 of theirs take no bits from them: at the start,
    in the middle and at the end, in tiles with the others."""
    n = 300
    q = torch.randn(q_len, heads * d, generator=_gen(1))
    q.view(q_len, heads, d)[..., 0] = 8.0
    k, v = (torch.randn(n, kv_heads, d, generator=_gen(i)) for i in (2, 3))
    large = torch.tensor([0, 5, 131, 160, n - q_len])
    k[large, :, 0] = -48.0 * d**0.5 / 8.0
    v[large] *= 2.0**far
    cache, seqs = _cache(k, v, page)
    q = q.bfloat16().cuda()
    out = _attend(cache, seqs, n, q, room, q_len=q_len)
    _check(cache, seqs, n, q, out, heads, q_len, groups=range(d // 32))


@pytest.mark.parametrize("d,heads,kv_heads,q_len,page", SHAPES[1:5])
@pytest.mark.parametrize("less", [8, 12, 16, 18])
@pytest.mark.parametrize("room", [0, 1 << 17])
def test_small_groups_beside_large_ones(d, heads, kv_heads, q_len, page, less, room):
    """A group of 32 dims whose values are 2^-less of its neighbours' is right by itself."""
    n = 200
    q = torch.randn(q_len, heads * d, generator=_gen(1)).bfloat16().cuda()
    k, v = (torch.randn(n, kv_heads, d, generator=_gen(i)) for i in (2, 3))
    v[..., 32:64] *= 2.0**-less
    v[..., 32:64] += 2.0**-less  # (an output that is not only what is left of a sum)
    cache, seqs = _cache(k, v, page)
    out = _attend(cache, seqs, n, q, room, q_len=q_len)
    _check(cache, seqs, n, q, out, heads, q_len, groups=range(d // 32))


@pytest.mark.parametrize("d,heads,kv_heads,q_len,page", SHAPES)
@pytest.mark.parametrize("size", [2.0**-66, 2.0**-40, 2.0**40, 2.0**90])
@pytest.mark.parametrize("room", [0, 1 << 17])
def test_values_of_any_size(d, heads, kv_heads, q_len, page, size, room):
    n = 150
    q = torch.randn(q_len, heads * d, generator=_gen(1)).bfloat16().cuda()
    k, v = (torch.randn(n, kv_heads, d, generator=_gen(i)) for i in (2, 3))
    cache, seqs = _cache(k, v * size, page)
    out = _attend(cache, seqs, n, q, room, q_len=q_len)
    _check(cache, seqs, n, q, out, heads, q_len)


@pytest.mark.parametrize("d,heads,kv_heads,q_len,page", SHAPES)
@pytest.mark.parametrize("size", [1.0, 2.0**20, 2.0**45])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 5)])
def test_zeros_count_in_the_sum(d, heads, kv_heads, q_len, page, size, window, sinks):
    """Tokens without a value have their weights, however large the others' values are; with a window some large ones are seen by a
    row and not by the next, or by none."""
    n = 250
    q = torch.randn(q_len, heads * d, generator=_gen(1)).bfloat16().cuda()
    k, v = (torch.randn(n, kv_heads, d, generator=_gen(i)) for i in (2, 3))
    v = v * size
    v[torch.rand(n, generator=_gen(4)) < 0.6] = 0.0
    v[160:162] *= 2.0**10
    cache, seqs = _cache(k, v, page)
    for room in (0, 1 << 17):
        out = _attend(cache, seqs, n, q, room, q_len=q_len, window=window, sinks=sinks)
        _check(cache, seqs, n, q, out, heads, q_len, window, sinks)


@pytest.mark.parametrize("d", [32, 64, 128])
def test_results_do_not_depend_on_how_a_sequence_is_cut(d):
    """One CTA, clusters and stretches: the same weights up to their rounding, with tokens of all sizes."""
    n, page, heads = 3000, 64, 4
    q = torch.randn(1, heads * d, generator=_gen(1)).bfloat16().cuda()
    k, v = (torch.randn(n, 1, d, generator=_gen(i)) for i in (2, 3))
    v *= torch.exp2(torch.randint(-30, 31, (n, 1, 1), generator=_gen(4)).float())
    cache, seqs = _cache(k, v, page)
    outs = [_attend(cache, seqs, n, q, room) for room in (0, 1 << 14, 1 << 17, 1 << 20)]
    for out in outs:
        _check(cache, seqs, n, q, out, heads, 1)
