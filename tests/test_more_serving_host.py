"""What the 4-bit cache, the reading of a cache and the packed attention decide before a launch (no GPU)."""

import ctypes
import math
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import serving_fp64 as oracle
from test_serving_host import _On, library  # noqa: F401 (a fixture)
from tiktoktechjam2026track3_b200 import _capi, packed_attention, serving
from tiktoktechjam2026track3_b200.build import build

HEADER = Path(__file__).resolve().parents[1] / "include" / "b200tx.h"
P, ODD, HUGE = 256, 264, (1 << 63) - 8  # addresses that nobody looks at: every call is refused, or has nothing to do


@pytest.fixture(scope="module")
def lib():
    build()
    return _capi.load_library()


def _call(fn, layout, *args):
    return fn(layout.pack(*(0 if a is None else a for a in args)), None)


# ---------------------------------------------------------------------------------- the formula of a step
def test_two_products_divide_by_fifteen():
    """A step is the range over 15: the range times the rounded 1 / 15, and its remainder times the same once more, is the
    rounded quotient for every mantissa (whole numbers in place of fp32, all 2^23 of them)."""
    k = int(float(np.float32(1) / np.float32(15)) * 2**27)
    x = np.arange(2**23, 2**24, dtype=np.int64)

    def rounded(v):  # to 24 bits, to the even one at a half
        e = np.floor(np.log2(v.astype(np.float64))).astype(np.int64)
        e += (v >> (e + 1) > 0).astype(np.int64) - (v >> e == 0).astype(np.int64)
        s = np.maximum(e - 23, 0)
        low, f = v & ((1 << s) - 1), v >> s
        half = np.where(s > 0, 1 << np.maximum(s - 1, 0), 1 << 62)
        return (f + ((low > half) | ((low == half) & (f & 1 == 1)))) << s

    q = rounded(x * k)                    # in 2^-27
    rest = (x << 27) - 15 * q             # exact, and fp32 holds it: a multiple of 2^22 below 2^8 of them
    assert not (q % 2**22).any() and not (rest % 2**22).any() and np.abs(rest // 2**22).max() < 256
    got = rounded(((q // 2**22) << 27) + rest // 2**22 * k)  # in 2^-32
    whole = (x << 32) // 15
    exact = rounded(2 * whole + ((x << 32) > 15 * whole))    # in 2^-33, with what is left in the lowest bit
    assert np.array_equal(2 * got, exact)


def test_the_reciprocal_of_a_step_is_far_from_a_border():
    """1 / step of a bf16 step lies at least 2^-17 of itself from the middle between two bf16 values (or is one): an approximate
    reciprocal, within 2^-22, rounds to the same."""
    for m in range(128, 256):
        x = 2.0**15 / m  # in (128, 256]
        border = math.floor(x) + 0.5
        assert abs(x - border) >= 2.0**-17 * x


def test_what_four_bits_hold():
    """The oracle's own arithmetic: codes decode to the values, halves go to the even code, odd groups."""
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(5, 3, 96, generator=g) * 4).bfloat16()
    step, mid = oracle.int4_params(x)
    y = oracle.int4(x)
    assert bool(((y - x.double()).abs() <= 0.55 * step.repeat_interleave(32, -1) + 2**-8 * mid.repeat_interleave(32, -1).abs()).all())
    codes = torch.round(((y.view(5, 3, 3, 32) - mid[..., None]) / step[..., None])).long() + 8
    bytes_ = torch.zeros(5, 3, 48, dtype=torch.uint8)
    for d in range(96):
        group, i = divmod(d, 32)
        at = 2 * ((i // 4) * 3 + group) + (i % 4) // 2
        bytes_[..., at] |= (codes[..., group, i] << (4 * (i % 2))).to(torch.uint8)
    params = torch.stack([step, mid], -2).bfloat16()
    assert torch.equal(oracle.int4_decode(bytes_, params), y)
    flat = torch.zeros(1, 32)
    assert torch.equal(oracle.int4(flat + 3), flat.double() + 3) and torch.equal(oracle.int4(flat), flat.double())
    flat[0, 3] = math.inf
    assert bool(torch.isnan(oracle.int4(flat)).all())


# ---------------------------------------------------------------------------------- refusals of the library
def _int4(**changes):
    fields = dict(k=256, v=256, pages=8, kv_heads=2, page_size=32, head_dim=64, page_stride=2 * 32 * 64, head_stride=32 * 64,
                  dtype=_capi.CACHE_INT4, k_group=256, v_group=256)
    return _capi.KVCacheDesc(**(fields | changes))


def _read(lib, cache, out_start=P, length=P, start=P, batch=2, pages=P, table_pages=2, most=4, rows=4, k=P, ld_k=128, v=P, ld_v=128):
    return _call(lib.b2_cache_read_fwd, _capi.CACHE_READ_ARGS, cache and ctypes.addressof(cache), out_start, length, start, batch,
                 pages, table_pages, most, rows, k, ld_k, v, ld_v)


@pytest.mark.parametrize("change,status", [
    (dict(k=None), 1), (dict(k_group=None), 1), (dict(v_group=None), 1), (dict(k_group=264), 2), (dict(head_dim=48), 2),
    (dict(head_dim=16), 2), (dict(head_dim=288, page_stride=1 << 15, head_stride=1 << 14), 2), (dict(page_size=8), 2),
    (dict(page_stride=2 * 32 * 64 - 32), 1), (dict(head_stride=32 * 64 + 16, page_stride=3 * 32 * 64), 2),
    (dict(page_stride=2 * 32 * 64 + 16), 2), (dict(head_stride=1 << 62), 1), (dict(v=264), 2)])
def test_bad_caches_are_rejected(lib, change, status):
    c = _int4(**change)
    at = ctypes.addressof(c)
    assert _read(lib, c) == status
    assert _call(lib.b2_cache_append_fwd, _capi.CACHE_APPEND_ARGS, at, P, 512, 0, 256, 384, 4, 4, 1, P, P, P, P, 2, 4, P, 64, 64, 0,
                 P, 256, None, 0) == status
    assert _call(lib.b2_cache_attention_fwd, _capi.CACHE_ATTENTION_ARGS, at, P, 256, 1, 1, 4, P, 2, P, 0, 0, 0.125, P, 256, P,
                 1 << 30) == status


def test_caches_of_other_types_need_no_groups(lib):
    """Their struct may be an older one, that ends before the groups: nothing is asked of them."""
    for dtype, scale in ((_capi.CACHE_BF16, None), (_capi.CACHE_E4M3, 256)):
        c = _int4(dtype=dtype, k_scale=scale, v_scale=scale, k_group=3, v_group=5)
        assert _read(lib, c, rows=0) == 0


def test_cache_read_rejects_bad_arguments(lib):
    c = _int4()
    assert _read(lib, None) == 1 and lib.b2_cache_read_fwd(None, None) == 1
    for name in ("out_start", "length", "start", "pages"):
        assert _read(lib, c, **{name: None}) == 1, name
    assert _read(lib, c, k=None, v=None) == 1
    assert _read(lib, c, batch=-1) == 1 and _read(lib, c, rows=-1) == 1 and _read(lib, c, most=-1) == 1
    assert _read(lib, c, table_pages=0) == 1 and _read(lib, c, table_pages=1 << 40) == 2
    assert _read(lib, c, batch=70000) == 2 and _read(lib, c, rows=HUGE) == 2 and _read(lib, c, most=HUGE) == 2
    assert _read(lib, c, ld_k=120) == 2 and _read(lib, c, ld_v=132) == 2 and _read(lib, c, k=ODD) == 2 and _read(lib, c, v=ODD) == 2
    assert _read(lib, c, batch=0) == 0 and _read(lib, c, rows=0) == 0 and _read(lib, c, most=0) == 0
    assert _read(lib, c, rows=0, k=None, ld_k=0) == 0


def test_packed_attention_rejects_bad_arguments(lib):
    def call(q=P, ld_q=256, rows=100, k=P, ld_k=128, v=P, ld_v=128, kv_rows=300, q_start=P, kv_start=P, batch=2, heads=4, kv_heads=2,
             head_dim=64, window=10, sinks=2, scale=0.125, out=P, ld_out=256):
        return _call(lib.b2_packed_attention_fwd, _capi.PACKED_ATTENTION_ARGS, q, ld_q, rows, k, ld_k, v, ld_v, kv_rows, q_start,
                     kv_start, batch, heads, kv_heads, head_dim, window, sinks, scale, out, ld_out)

    assert lib.b2_packed_attention_fwd(None, None) == 1
    for name in ("q", "k", "v", "out"):
        assert call(**{name: None}) == 1, name
        assert call(**{name: ODD + 2}) == 2, name
    assert call(q_start=None) == 1 and call(kv_start=None) == 1
    assert call(heads=3) == 1 and call(kv_heads=0) == 1 and call(batch=-1) == 1 and call(rows=-1) == 1 and call(kv_rows=-1) == 1
    for scale in (0.0, -1.0, math.nan, math.inf, 1e300, 1e-300):
        assert call(scale=scale) == 1, scale
    assert call(window=-1) == 1 and call(sinks=-1) == 1 and call(window=0) == 1  # sinks without a window
    assert call(head_dim=48) == 2 and call(head_dim=256, ld_q=1024, ld_k=512, ld_v=512, ld_out=1024) == 2
    assert call(ld_q=248) == 1 and call(ld_k=120) == 1 and call(ld_v=120) == 1 and call(ld_out=248) == 1 and call(ld_out=257) == 2
    assert call(rows=1 << 29) == 2 and call(kv_rows=1 << 29) == 2 and call(batch=1 << 21) == 2 and call(heads=1 << 62) == 2
    assert call(heads=1 << 58, kv_heads=1 << 57) == 2 and call(ld_k=HUGE) == 2 and call(heads=70000, kv_heads=1, ld_q=HUGE) == 2
    assert call(batch=0) == 0 and call(rows=0) == 0 and call(rows=0, kv_rows=0, k=None, v=None) == 0


def test_argument_structs_have_the_headers_layout():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    for name, layout in (("cache_read", _capi.CACHE_READ_ARGS), ("packed_attention", _capi.PACKED_ATTENTION_ARGS)):
        body = re.search(r"typedef struct b2_%s_args \{(.*?)\}" % name, text, flags=re.S).group(1)
        kinds = "".join(("d" if line.startswith("double") else "q") * len(line.split(","))
                        for line in filter(None, (part.strip() for part in body.split(";"))))
        assert kinds == "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([qd])", layout.format)), name
    body = re.search(r"typedef struct b2_kv_cache \{(.*?)\}", text, flags=re.S).group(1)
    members = [m.strip(" *") for line in body.split(";") if line.strip() for m in re.sub(r"^(void|float|int64_t|int)\b", "", line.strip()).split(",")]
    assert members == [name for name, _ in _capi.KVCacheDesc._fields_]


# ---------------------------------------------------------------------------------- refusals of the wrappers
def _calls(device):
    i32 = torch.int32
    desc = _capi.KVCacheDesc(pages=4, kv_heads=2, page_size=16, head_dim=64)
    desc.device = device

    def on(*shape, dtype=torch.bfloat16):
        return _On(device, shape, dtype)

    return {
        "b2_cache_read_fwd": (_capi.cache_read, dict(
            out_start=on(2, dtype=i32), length=on(2, dtype=i32), start=on(2, dtype=i32), page_table=on(2, 3, dtype=i32),
            k_out=on(5, 128), v_out=on(5, 128)), dict(cache=desc, max_len=4)),
        "b2_packed_attention_fwd": (_capi.packed_attention, dict(
            q=on(6, 256), k=on(9, 128), v=on(9, 128), q_start=on(3, dtype=i32), kv_start=on(3, dtype=i32), out=on(6, 256)),
            dict(head_dim=64, window=0, sinks=0, scale=0.1)),
    }


@pytest.mark.parametrize("device", [0, 1])
def test_calls_run_on_the_gpu_of_their_tensors(library, device):  # noqa: F811
    for name, (call, tensors, rest) in _calls(device).items():
        call(**tensors, **rest)
        assert library.calls.pop() == (name, device, 100 + device)
    assert _capi._current_device() == 0


def test_tensors_of_another_gpu_are_refused(library):  # noqa: F811
    for call, tensors, rest in _calls(0).values():
        for name, t in tensors.items():
            with pytest.raises(ValueError, match="must be on cuda"):
                call(**(tensors | {name: _On(1, t.shape, t.dtype)}), **rest)
    assert not library.calls


def test_shapes_and_types_that_do_not_fit_are_refused(library):  # noqa: F811
    for call, tensors, rest in _calls(0).values():
        for name, t in tensors.items():
            for bad in (_On(0, t.shape, torch.float32), _On(0, (*t.shape[:-1], t.shape[-1] + 1), t.dtype),
                        _On(0, (t.shape[0] + 1, *t.shape[1:]), t.dtype)):
                if name in ("q_start", "page_table") and bad.dtype == t.dtype and (name != "page_table" or bad.shape[0] == t.shape[0]):
                    continue  # (another number of sequences; a wider table)
                with pytest.raises(ValueError):
                    call(**(tensors | {name: bad}), **rest)
        for name in {"window", "sinks", "max_len"} & set(rest):
            for bad in (4.0, 1 << 70):
                with pytest.raises(TypeError, match="integers"):
                    call(**tensors, **(rest | {name: bad}))
    call, tensors, rest = _calls(0)["b2_packed_attention_fwd"]
    for bad in (dict(head_dim=0), dict(head_dim=-64), dict(head_dim=96)):
        with pytest.raises(ValueError, match="heads"):
            call(**tensors, **(rest | bad))
    with pytest.raises(ValueError, match="q_start"):
        call(**(tensors | dict(q_start=_On(0, (0,), torch.int32))), **rest)
    call, tensors, rest = _calls(0)["b2_cache_read_fwd"]
    with pytest.raises(ValueError, match="needed"):
        call(**(tensors | dict(k_out=None, v_out=None)), **rest)
    assert not library.calls


def test_caches_that_are_none_are_refused():
    for head_dim in (0, -32, 16, 33, 80):
        with pytest.raises(ValueError, match="multiple of 32"):
            serving.KVCache.allocate(2, 1, head_dim, 16, torch.uint8, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        serving.KVCache.allocate(2, 1, 64, 16, torch.uint8, device="cpu")
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        packed_attention(x, x, x, torch.zeros(2, dtype=torch.int32), None, 64)


def test_kernels_read_a_cache_past_the_read_only_path():
    """The launch that writes codes and parameters may still run when a reader's first CTAs are resident; only tables of
    positions, which no kernel writes, come by it."""
    text = (Path(serving.__file__).parent / "csrc" / "cache_int4.cuh").read_text()
    assert "pdl_wait_previous_grid" in text
    assert not re.search(r"ld\.global(\.\w+)*\.nc", text)
    assert all("row" in line for line in text.splitlines() if "__ldg" in line)
