"""Starts of packed sequences that do not ascend, or lie outside the rows, on a B200: whose rows are computed, and that others' are
not touched. The rows themselves are compared with the same call of that sequence alone, bit for bit."""

import random

import pytest
import torch

from test_gpu_packed import BF16, _gen, _i32
from tiktoktechjam2026track3_b200 import _capi, serving

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_status(cuda_device):
    _capi.device_status(clear=True)
    yield
    torch.cuda.synchronize()
    assert _capi.device_status(clear=True) == 0


def _valid(q_at, kv_at, rows, keys):
    """The sequences that are computed: inside the rows, not ending before they begin, and not beginning before an earlier start that
    lies inside the rows."""
    most, valid = -1, []
    for b in range(len(q_at) - 1):
        inside = 0 <= q_at[b] <= rows
        valid.append(inside and q_at[b] >= most and q_at[b] <= q_at[b + 1] <= rows and 0 <= kv_at[b] <= kv_at[b + 1] <= keys)
        if inside:
            most = max(most, q_at[b])
    return valid


def _run(q_at, kv_at, rows, keys, heads, kv_heads, d, window=0, sinks=0, many=False):
    q = torch.randn(rows, heads * d, generator=_gen(1)).bfloat16().cuda()
    k, v = (torch.randn(keys, kv_heads * d, generator=_gen(i)).bfloat16().cuda() for i in (2, 3))
    out = torch.full_like(q, 9.0)
    args = dict(window=window, sinks=sinks)
    serving.packed_attention(q, k, v, _i32(q_at), _i32(kv_at), d, out=out, **args)
    torch.cuda.synchronize()
    assert _capi.device_status(clear=True) == (9 << 16) | (1 << 8) | 3
    want = torch.full_like(q, 9.0)
    done = out == 9.0
    for b, valid in enumerate(_valid(q_at, kv_at, rows, keys)):
        if valid or (many and 0 <= q_at[b] <= q_at[b + 1] <= rows):
            own, kv = slice(q_at[b], q_at[b + 1]), slice(kv_at[b], kv_at[b + 1])
            serving.packed_attention(q[own], k[kv], v[kv], _i32([0, q_at[b + 1] - q_at[b]]), _i32([0, kv_at[b + 1] - kv_at[b]]), d,
                                     out=want[own], **args)
            done[own] |= out[own] == want[own]
    if many:  # some may be skipped with the bad one, and values that two claim are either's
        assert bool(done.all())
    else:
        assert torch.equal(out, want)


BAD = [
    ([0, 1000, -1, 2000], 2000),
    ([0, 1000, 0, 2000], 2000),
    ([0, 1000, 2000, -5, 2100, 2500], 2500),
    ([0, 1000, 1000, 1200, 5, 1500], 1500),
    ([0, 700, 300, 1500, 1500, 1900], 1900),       # 300 ... 1500 begins before 700
    ([0, 400, 5000, 900, 1300], 1300),              # beyond the rows
    ([0, 400, 1300, 900, 1300], 1300),              # inside them: the second sequence reaches to the end
    ([-7, 300, 600], 600),
    ([600, 0, 300], 600),
    ([0, 2**31 - 1, -2**31, 500, 900], 900),
    ([0, 130, 257, 257, 256, 600, 900, 899, 1400, 1400, 3, 1800], 1800),
]


@pytest.mark.parametrize("q_at,rows", BAD)
@pytest.mark.parametrize("heads,kv_heads,d", [(1, 1, 64), (4, 1, 128), (16, 1, 32), (3, 1, 64)])
def test_a_bad_start_takes_no_rows_from_others(q_at, rows, heads, kv_heads, d):
    """Several query tiles to a sequence: each of the valid ones is computed whole, whatever start stands behind it."""
    kv_at = [600 * b for b in range(len(q_at))]
    _run(q_at, kv_at, rows, kv_at[-1], heads, kv_heads, d)


@pytest.mark.parametrize("d,window,sinks", [(64, 0, 0), (128, 100, 20)])
def test_bad_starts_of_keys(d, window, sinks):
    """A start of keys is no place of a query tile: only the sequences that it bounds are skipped."""
    q_at = [0, 400, 800, 1300, 1301]
    for kv_at in ([0, 500, -1, 1500, 1600], [0, 500, 300, 1500, 1600], [0, 500, 1601, 1500, 1600], [-1, 500, 900, 1500, 1601]):
        _run(q_at, kv_at, 1301, 1600, 2, 1, d, window, sinks)


@pytest.mark.parametrize("seed", range(12))
def test_random_starts(seed):
    """Up to 32 sequences with some starts changed to anything."""
    rng = random.Random(seed)
    batch, rows = rng.randint(2, 32), rng.randint(300, 3000)
    q_at = [0] + sorted(rng.randint(0, rows) for _ in range(batch - 1)) + [rows]
    for _ in range(rng.randint(1, 3)):
        q_at[rng.randrange(batch + 1)] = rng.choice([-1, 0, rows, rows + 1, rng.randint(0, rows), -2**31, 2**31 - 1])
    kv_at = [37 * b for b in range(batch + 1)]
    if all(_valid(q_at, kv_at, rows, kv_at[-1])):
        q_at[1] = -1
    _run(q_at, kv_at, rows, kv_at[-1], 2, 1, 64)


@pytest.mark.parametrize("batch,at", [(33, 32), (40, 3), (100, 64), (1100, 32), (1100, 1024), (1100, 1099)])
@pytest.mark.parametrize("start", [-1, 0, 10, 10**9])
def test_a_bad_start_among_many(batch, at, start):
    """More sequences than a warp looks at at once: others may be skipped with it; each value is of a sequence that claims it."""
    q_at = [0]
    for b in range(batch):
        q_at.append(q_at[-1] + (40, 0, 130, 7, 64)[b % 5])
    rows = q_at[-1]
    kv_at = [5 * b for b in range(batch + 1)]
    q_at[at] = start
    _run(q_at, kv_at, rows, kv_at[-1], 1, 1, 64, many=True)
