"""The 4-bit cache, reading a cache back and the packed attention where calls, memory and odd values meet, on a B200.

Tolerances are those of test_gpu_int4.py and test_gpu_packed.py.
"""

import math

import pytest
import torch

from test_gpu_int4 import BF16, E4M3, INT4, _check_attend, _decode, _filled, _gen, _i32, _of, _Sequences, _starts
from test_gpu_packed import _check as _check_packed
from oracle import serving_fp64 as oracle
from tiktoktechjam2026track3_b200 import _capi, serving

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_status(cuda_device):
    _capi.device_status(clear=True)
    yield
    torch.cuda.synchronize()
    assert _capi.device_status(clear=True) == 0


def _wide(seqs, page, room=1 << 17):
    """The page table with columns for `room` tokens: heads are then cut into stretches, which need the workspace."""
    return torch.nn.functional.pad(seqs.table, (0, room // page - seqs.table.shape[1]), value=-1).cuda()


def _randn(seed, *shape):
    return torch.randn(*shape, generator=_gen(seed)).bfloat16().cuda()


# ---------------------------------------------------------------------------------- codes at the ends of their range
@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
def test_groups_far_from_zero_next_to_others(d):
    """A middle that is rounded by steps takes codes beyond 0 ... 15 for some groups of a warp's tokens and not for others:
    each ends where the range does. What is stored is compared bit for bit, as anywhere without a rotation."""
    kv_heads, n = 3, 61
    x = torch.randn(n, 2 * kv_heads, d // 32, 32, generator=_gen(d))
    far = torch.randint(0, 3, (n, 2 * kv_heads, d // 32, 1), generator=_gen(1)) == 0
    x = (x + far * torch.randn(far.shape, generator=_gen(2)) * 3000).bfloat16().view(n, 2 * kv_heads, d)
    step, mid = oracle.int4_params(x)
    by = ((x.double().view(n, 2 * kv_heads, -1, 32).amin(-1) - mid) / step).nan_to_num()
    assert bool((by < -9).any()) and bool((by > -7).any())  # (codes that would lie below 0, and ranges that begin above it)
    seqs = _Sequences([n], 16, 3)
    cache = serving.KVCache.allocate(seqs.pages, kv_heads, d, 16, INT4)
    qkv = torch.cat([torch.zeros(n, kv_heads * d, dtype=BF16), x.flatten(1)], 1).cuda()
    cache.append(qkv, kv_heads, _i32([0]), _i32([n]), _i32([0]), seqs.table.cuda(), n)
    for which, given in (("k", x[:, :kv_heads]), ("v", x[:, kv_heads:])):
        got = _of(_decode(cache, which), seqs.table[0], 16, 0, n)
        assert torch.equal(got.transpose(0, 1), oracle.int4(given))


@pytest.mark.parametrize("dtype", [INT4, E4M3, BF16])
@pytest.mark.parametrize("d,rotary_dim,interleaved,heads", [(64, 64, False, 2), (128, 32, True, 4), (96, 96, False, 3)])
def test_a_table_that_begins_between_two_32_byte_blocks(dtype, d, rotary_dim, interleaved, heads):
    """Tables need 16-byte alignment only; how they are loaded does not change a result."""
    table = serving.rotary_table(128, rotary_dim)
    room = torch.zeros(table.numel() + 4, device="cuda")
    off = room[4:].view(table.shape)
    off.copy_(table)
    assert table.data_ptr() % 32 == 0 and off.data_ptr() % 32 == 16
    qkv = _randn(4, 50, (heads + 2) * d)
    seqs = _Sequences([50], 32, 1)
    outs = []
    for t in (table, off):
        cache = serving.KVCache.allocate(seqs.pages, 1, d, 32, dtype)
        q = cache.append(qkv, heads, _i32([0]), _i32([50]), _i32([0]), seqs.table.cuda(), 50, table=t, interleaved=interleaved)
        turned = serving.rotary(qkv[:, :heads * d], torch.arange(50, dtype=torch.int32, device="cuda"), t, d,
                                interleaved=interleaved)
        assert torch.equal(q, turned)
        outs.append((q, cache.k.view(torch.uint8), cache.v.view(torch.uint8)))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------------- memory
def test_pages_that_are_slices_of_one_buffer():
    """K and V side by side in a page, with room between heads: strides of the caller's."""
    lengths, page, hk, d = [70, 33], 32, 2, 64
    seqs = _Sequences(lengths, page, 2)
    buffer = torch.randint(0, 256, (seqs.pages, 2, hk, page + 16, d // 2), generator=_gen(1), dtype=torch.uint8).cuda()
    groups = [torch.full((seqs.pages, hk, page, 2, d // 32), math.nan, dtype=BF16, device="cuda") for _ in range(2)]
    cache = serving.KVCache(buffer[:, 0, :, :page], buffer[:, 1, :, :page], *groups)
    plain = serving.KVCache.allocate(seqs.pages, hk, d, page, INT4)
    before = buffer.clone()
    qkv = _randn(3, sum(lengths), 4 * hk * d)
    step = (2 * hk, _i32(_starts(lengths)), _i32(lengths), _i32([0, 0]), seqs.table.cuda(), 70)
    q = qkv[:2, :2 * hk * d]
    outs = []
    for c in (cache, plain):
        c.append(qkv, *step)
        k, v = (torch.empty(103, hk * d, dtype=BF16, device="cuda") for _ in range(2))
        c.read(_i32([0, 70]), _i32(lengths), _i32([0, 0]), seqs.table.cuda(), 70, k_out=k, v_out=v)
        outs.append((k, v, c.attend(q, seqs.table.cuda(), _i32(lengths)), c.attend(q, _wide(seqs, page), _i32(lengths))))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert torch.equal(buffer[:, :, :, page:], before[:, :, :, page:])


def test_pages_more_than_32_bits_away():
    """5 GB of codes each for keys and values: the last pages, for all three operators."""
    page, d, pages = 256, 128, 310_000
    codes = [torch.zeros(pages, 1, page, d // 2, dtype=torch.uint8, device="cuda") for _ in range(2)]
    groups = [torch.zeros(pages, 1, page, 2, d // 32, dtype=BF16, device="cuda") for _ in range(2)]
    cache = serving.KVCache(*codes, *groups)
    small = serving.KVCache.allocate(3, 1, d, page, INT4)
    n = 700
    qkv, q = _randn(1, n, 3 * d), _randn(2, 1, 4 * d)
    outs = []
    for c, table in ((cache, [[pages - 1, pages - 3, pages - 2]]), (small, [[2, 0, 1]])):
        table = _i32(table)
        c.append(qkv, 1, _i32([0]), _i32([n]), _i32([0]), table, n)
        k, v = (torch.zeros(n, d, dtype=BF16, device="cuda") for _ in range(2))
        c.read(_i32([0]), _i32([n]), _i32([0]), table, n, k_out=k, v_out=v)
        wide = torch.nn.functional.pad(table, (0, 509), value=-1)
        outs.append((k, v, c.attend(q, table, _i32([n])), c.attend(q, wide, _i32([n]))))
    for a, b in zip(*outs):
        assert torch.equal(a, b) and bool(a.any())
    assert not bool(codes[0][:1000].any())


@pytest.mark.parametrize("d,heads,kv_heads", [(32, 4, 2), (64, 16, 2), (128, 20, 1)])
@pytest.mark.parametrize("room", [0, 1 << 17])
def test_parameters_of_tokens_that_no_row_sees_are_not_used(d, heads, kv_heads, room):
    """NaN and infinities behind the last token, between sinks and window, and in page 0, which nobody owns (tiles that are
    missing at a sequence's end read it)."""
    lengths, page, window, sinks = [300, 17, 90], 16, 40, 5
    cache, seqs = _filled(lengths, page, kv_heads, d, INT4, 9)
    if bool((seqs.table == 0).any()):
        free = next(i for i in range(seqs.pages - 1, 0, -1) if not bool((seqs.table == i).any()))
        for x in (cache.k, cache.v, cache.k_scale, cache.v_scale):
            x[free] = x[0]
        seqs.table[seqs.table == 0] = free
    for x in (cache.k_scale, cache.v_scale):
        x[0] = math.inf
        for b, n in enumerate(lengths):  # tokens behind the sinks and before every row's window
            for j in range(sinks, max(sinks, n - window)):
                x[int(seqs.table[b, j // page]), :, j % page] = -math.inf if j % 2 else math.nan
    table = _wide(seqs, page, room) if room else seqs.table.cuda()
    q = _randn(1, 3, heads * d)
    out = cache.attend(q, table, _i32(lengths), window=window, sinks=sinks)
    kept = serving.KVCache(cache.k, cache.v, cache.k_scale.nan_to_num(0.0, 0.0, 0.0), cache.v_scale.nan_to_num(0.0, 0.0, 0.0))
    _check_attend(kept, seqs, lengths, heads, 1, window, sinks, q, out, d**-0.5)


def test_a_group_that_is_not_finite_reaches_the_rows_that_see_it():
    lengths, page, d = [64], 16, 64
    cache, seqs = _filled(lengths, page, 1, d, INT4, 1)
    cache.v_scale[int(seqs.table[0, 1]), 0, 3, :, 1] = math.nan  # token 19, elements 32 ...
    q = _randn(1, 1, d)
    out = cache.attend(q, seqs.table.cuda(), _i32(lengths))
    assert bool(torch.isnan(out[0, 32:]).all()) and bool(torch.isfinite(out[0, :32]).all())
    q[0, 0] = math.inf
    assert not bool(torch.isfinite(cache.attend(q, seqs.table.cuda(), _i32(lengths))).any())


@pytest.mark.parametrize("d,heads,kv_heads,page", [(32, 2, 1, 16), (64, 4, 2, 16), (64, 12, 1, 32), (64, 2, 2, 128), (128, 8, 1, 16),
                                                   (128, 4, 4, 64), (32, 12, 1, 32)])
@pytest.mark.parametrize("window,sinks,q_len", [(40, 4, 1), (100, 0, 2), (33, 70, 1), (1, 1, 1)])
@pytest.mark.parametrize("room", [0, 1 << 17])
def test_pages_that_no_row_sees_need_not_be_there(d, heads, kv_heads, page, window, sinks, q_len, room):
    """Pages between the sinks and the window given back, as a streaming cache does: -1, or past the cache, in the table."""
    lengths = [700, 333, 90]
    cache, seqs = _filled(lengths, page, kv_heads, d, INT4, 9)
    table = _wide(seqs, page, room) if room else seqs.table.cuda()
    q = _randn(1, 3 * q_len, heads * d)
    args = dict(window=window, sinks=sinks, q_len=q_len)
    want = cache.attend(q, table, _i32(lengths), **args)
    _check_attend(cache, seqs, lengths, heads, q_len, window, sinks, q, want, d**-0.5)
    gone = 0
    for b, n in enumerate(lengths):
        for i in range(-(-n // page)):
            if i * page >= sinks and (i + 1) * page <= n - q_len - window + 1:
                table[b, i] = -1 if i % 2 else cache.pages + 5
                gone += 1
    assert gone
    assert torch.equal(cache.attend(q, table, _i32(lengths), **args), want)


def test_attend_with_a_scale_that_hides_nothing():
    """Scales at the small end, where all weights are alike, and queries of zeros."""
    lengths, d = [100, 17], 64
    cache, seqs = _filled(lengths, 16, 1, d, INT4, 3)
    mean = [_of(_decode(cache, "v"), seqs.table[b], 16, 0, n)[0].mean(0) for b, n in enumerate(lengths)]
    for q, scale in ((_randn(1, 2, d), 1e-40), (torch.zeros(2, d, dtype=BF16, device="cuda"), 1e-40),
                     (torch.zeros(2, d, dtype=BF16, device="cuda"), 1.0), (_randn(1, 2, d) * 2.0**-110, 1e-20)):
        out = cache.attend(q, seqs.table.cuda(), _i32(lengths), scale=scale).cpu().double()
        for b in range(2):
            assert bool(((out[b] - mean[b]).abs() <= 2**-8 * mean[b].abs() + 2**-9 * 8).all())


# ---------------------------------------------------------------------------------- calls
@pytest.mark.parametrize("heads,kv_heads,d,q_len", [(16, 1, 64, 5), (40, 2, 128, 27), (12, 1, 32, 47)])
def test_attend_with_many_row_blocks(heads, kv_heads, d, q_len):
    lengths = [1100, 30, 3000]
    cache, seqs = _filled(lengths, 64, kv_heads, d, INT4, 8)
    q = _randn(2, len(lengths) * q_len, heads * d)
    outs = [cache.attend(q, table, _i32(lengths), q_len=q_len) for table in (seqs.table.cuda(), _wide(seqs, 64)) for _ in range(2)]
    for out in outs[::2]:
        _check_attend(cache, seqs, lengths, heads, q_len, 0, 0, q, out, d**-0.5)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[2], outs[3])


def test_one_workspace_for_caches_of_any_type():
    lengths = [4000] + [70 + 5 * b for b in range(63)]
    caches = [_filled(lengths, 64, 2, 64, INT4, 1), _filled(lengths, 64, 1, 128, BF16, 2), _filled(lengths, 32, 1, 128, INT4, 3)]
    calls = []
    for cache, seqs in caches:
        table = _wide(seqs, cache.page_size)
        for batch, q_len in ((1, 16), (64, 1), (3, 4), (64, 2), (1, 1)):
            args = (_randn(batch, batch * q_len, 4 * cache.head_dim), table[:batch], _i32(lengths[:batch]))
            fresh = cache.workspace(batch, 4, q_len)
            calls.append((cache, args, q_len, cache.attend(*args, q_len=q_len, workspace=fresh)))
    shared = max((c.workspace(1, 4, 16) for c, _ in caches), key=lambda w: w.numel())
    for order in (calls, calls[::-1], calls[::2] + calls[1::2]):
        for cache, args, q_len, want in order:
            assert torch.equal(cache.attend(*args, q_len=q_len, workspace=shared), want)


@pytest.mark.parametrize("heads", [1, 8])
@pytest.mark.parametrize("room", [0, 1 << 17])
def test_steps_enqueued_at_once_are_those_waited_for_one_by_one(heads, room):
    """Append, attend and read in turn without a wait between: the same bits as with a wait after every call."""
    steps, d = 40, 64
    rows = (torch.randn(steps, 3 * heads * d, generator=_gen(11)) * torch.exp2(torch.arange(steps) / 3.0)[:, None]).bfloat16().cuda()
    got = []
    for wait in (False, True):
        cache = serving.KVCache.allocate(4, heads, d, 16, INT4)
        table = torch.nn.functional.pad(_i32([[2, 0, 3]]), (0, max(0, room // 16 - 3)), value=-1)
        past, lens = [_i32([i]) for i in range(steps)], [_i32([i + 1]) for i in range(steps)]
        zero, one = _i32([0]), _i32([1])
        back = [torch.zeros(steps, heads * d, dtype=BF16, device="cuda") for _ in range(2 * steps)]
        torch.cuda.synchronize()
        outs = []
        for i in range(steps):
            cache.append(rows[i:i + 1], heads, zero, one, past[i], table, 1)
            if wait:
                torch.cuda.synchronize()
            outs.append(cache.attend(rows[i:i + 1, :heads * d], table, lens[i]))
            if wait:
                torch.cuda.synchronize()
            cache.read(zero, lens[i], zero, table, i + 1, k_out=back[2 * i], v_out=back[2 * i + 1])
            if wait:
                torch.cuda.synchronize()
        got.append((torch.cat(outs), torch.stack(back)))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_a_captured_chunk_follows_its_lengths():
    """Append, read and packed attention in a graph: replayed with other rows, lengths, pages and positions, on another stream
    next to eager calls of the same kind."""
    batch, page, heads, hk, d, most = 3, 16, 4, 2, 64, 64
    pages = 12
    plans = [([20, 0, 9], [0, 5, 30]), ([1, 44, 3], [60, 0, 2]), ([16, 16, 16], [16, 32, 48])]

    def eager(cache, x, new, past, table):
        held = [p + n for p, n in zip(past, new)]
        q_at, kv_at = _starts(new), _starts(held)
        q_at, kv_at = q_at + [sum(new)], kv_at + [sum(held)]
        q = x[:, :heads * d]
        k, v, out = (torch.zeros(400, w * d, dtype=BF16, device="cuda") for w in (hk, hk, heads))
        cache.append(x, heads, _i32(q_at[:-1]), _i32(new), _i32(past), table, most)
        cache.read(_i32(kv_at[:-1]), _i32(held), _i32([0] * batch), table, 400, k_out=k, v_out=v)
        serving.packed_attention(q, k, v, _i32(q_at), _i32(kv_at), d, out=out[:x.shape[0]])
        return k, v, out

    table0 = torch.arange(batch * pages, dtype=torch.int32, device="cuda").view(batch, pages)
    caches = [serving.KVCache.allocate(batch * pages, hk, d, page, INT4) for _ in range(2)]
    x = torch.zeros(most, (heads + 2 * hk) * d, dtype=BF16, device="cuda")
    ints = dict(dtype=torch.int32, device="cuda")
    q_start, kv_start = torch.zeros(batch + 1, **ints), torch.zeros(batch + 1, **ints)
    new_len, past_len, held_len, zeros = (torch.zeros(batch, **ints) for _ in range(4))
    table = table0.clone()
    k, v, out = (torch.zeros(400, w * d, dtype=BF16, device="cuda") for w in (hk, hk, heads))

    def calls():
        caches[0].append(x, heads, q_start[:-1], new_len, past_len, table, most)
        caches[0].read(kv_start[:-1], held_len, zeros, table, 400, k_out=k, v_out=v)
        serving.packed_attention(x[:, :heads * d], k, v, q_start, kv_start, d, out=out[:most])

    calls()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        calls()
    for i, (new, past) in enumerate(plans):
        rows = _randn(i, most, (heads + 2 * hk) * d)
        pick = torch.randperm(batch * pages, generator=_gen(i)).int().view(batch, pages).cuda()
        held = [p + n for p, n in zip(past, new)]
        x.copy_(rows)
        table.copy_(pick)
        for t, values in ((q_start, _starts(new) + [sum(new)]), (kv_start, _starts(held) + [sum(held)]), (new_len, new),
                          (past_len, past), (held_len, held)):
            t.copy_(_i32(values))
        for buf in (k, v, out):
            buf.zero_()
        for name in ("k", "v", "k_scale", "v_scale"):
            getattr(caches[1], name).copy_(getattr(caches[0], name))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        want = eager(caches[1], rows, new, past, pick)
        torch.cuda.synchronize()
        for a, b in zip((k, v, out), want):
            assert torch.equal(a, b)
        for name in ("k", "v"):
            assert torch.equal(getattr(caches[0], name), getattr(caches[1], name))


def test_packed_attention_of_more_sequences_than_a_warp_looks_at_twice():
    """1100 sequences of up to 3 rows: three turns of the search."""
    new = [(7 * b) % 4 for b in range(1100)]
    past = [(5 * b) % 3 for b in range(1100)]
    q_at, kv_at = _starts(new) + [sum(new)], _starts([n + p for n, p in zip(new, past)]) + [sum(new) + sum(past)]
    q, k, v = _randn(1, q_at[-1], 2 * 32), _randn(2, kv_at[-1], 32), _randn(3, kv_at[-1], 32)
    out = serving.packed_attention(q, k, v, _i32(q_at), _i32(kv_at), 32)
    _check_packed(q, k, v, out, q_at, kv_at, 2, 1, 32, 0, 0)


@pytest.mark.parametrize("batch", [2, 31, 32, 33, 64])
@pytest.mark.parametrize("heads,kv_heads,d,window,sinks", [(1, 1, 64, 0, 0), (4, 1, 128, 0, 0), (16, 1, 32, 40, 5), (6, 2, 64, 0, 0)])
def test_packed_attention_of_many_unlike_sequences(batch, heads, kv_heads, d, window, sinks):
    """Empty ones, chunks behind many keys, more queries than keys: every tile of every sequence has its CTA, whichever way a
    CTA finds its own, and rows of no sequence stay as they are."""
    new = [(0, 1, 37, 128, 129, 16, 3)[(5 * b) % 7] for b in range(batch)]
    held = [max(0, n + (0, 300, -9, 0, 64, 1, -200)[(3 * b + b // 7) % 7]) for b, n in enumerate(new)]
    q_at, kv_at = [3], [2]
    for n, m in zip(new, held):
        q_at.append(q_at[-1] + n)
        kv_at.append(kv_at[-1] + m)
    q, k, v = _randn(1, q_at[-1] + 4, heads * d), _randn(2, kv_at[-1] + 1, kv_heads * d), _randn(3, kv_at[-1] + 1, kv_heads * d)
    out = torch.full_like(q, 9.0)
    serving.packed_attention(q, k, v, _i32(q_at), _i32(kv_at), d, window=window, sinks=sinks, out=out)
    _check_packed(q, k, v, out, q_at, kv_at, heads, kv_heads, d, window, sinks)
    assert bool((out[:3] == 9).all()) and bool((out[q_at[-1]:] == 9).all())


@pytest.mark.parametrize("batch", [6, 40])
def test_sequences_next_to_one_outside_the_rows(batch):
    """A start beyond the rows spoils the two sequences that it bounds; it is recorded, and the others are as they are alone."""
    new = [(40, 0, 130, 7, 64)[b % 5] for b in range(batch)]
    at = _starts(new) + [sum(new)]
    q, k, v = (_randn(i, at[-1], 64) for i in range(3))
    bad = list(at)
    bad[3] = at[-1] + 5
    want, got = (torch.full_like(q, 9.0) for _ in range(2))
    serving.packed_attention(q, k, v, _i32(at), _i32(at), 64, out=want)
    serving.packed_attention(q, k, v, _i32(bad), _i32(at), 64, out=got)
    torch.cuda.synchronize()
    assert _capi.device_status(clear=True) & 0xFF == _capi.REASON_BAD_INDEX
    for b in range(batch):
        rows = slice(at[b], at[b + 1])
        if b not in (2, 3):
            assert torch.equal(got[rows], want[rows])
        else:
            assert bool((got[rows] == 9).all())


def test_the_largest_strides_and_narrow_slices():
    """Rows far apart: one head of many columns, for keys, values and outputs alike."""
    rows, d, wide = 50, 64, 20_000
    big = torch.full((rows, wide), math.nan, dtype=BF16, device="cuda")
    q, k, v, out = (big[:, c:c + d] for c in (0, 4096, 8200, 19_000))
    for i, x in enumerate((q, k, v)):
        x.copy_(_randn(i, rows, d))
    serving.packed_attention(q, k, v, _i32([0, 20, rows]), None, d, out=out)
    _check_packed(q, k, v, out, [0, 20, rows], [0, 20, rows], 1, 1, d, 0, 0)
    cache = serving.KVCache.allocate(4, 1, d, 16, INT4)
    cache.append(big[:, 0:3 * d], 1, _i32([0]), _i32([0]), _i32([0]), _i32([[0, 1, 2, 3]]), 0)  # nothing new
    assert not bool(cache.k.any())


def test_indices_outside_their_tables_in_attend():
    cache, seqs = _filled([40], 16, 1, 64, INT4, 1)
    q = _randn(1, 1, 64)
    for table, n in ((seqs.table, 49), (seqs.table, -1), (torch.tensor([[99, -1, -1]], dtype=torch.int32), 40)):
        cache.attend(q, table.cuda(), _i32([n]))
        torch.cuda.synchronize()
        status = _capi.device_status(clear=True)
        assert status >> 16 == 7 and status & 0xFF == 3


@pytest.mark.parametrize("dtype", [INT4, E4M3, BF16])
def test_reading_what_is_there_twice_and_the_same_rows_twice(dtype):
    """Two sequences that share their pages, and one that is read from two places at once."""
    cache, seqs = _filled([100], 32, 2, 64, dtype, 4)
    table = seqs.table.repeat(3, 1).cuda()
    k, v = (torch.zeros(150, 128, dtype=BF16, device="cuda") for _ in range(2))
    cache.read(_i32([0, 100, 140]), _i32([100, 40, 10]), _i32([0, 60, 3]), table, 100, k_out=k, v_out=v)
    for which, out in (("k", k), ("v", v)):
        values = _decode(cache, which)
        parts = [_of(values, seqs.table[0], 32, a, b).transpose(0, 1).flatten(1) for a, b in ((0, 100), (60, 100), (3, 13))]
        assert torch.equal(out.cpu(), torch.cat(parts).float().bfloat16())
