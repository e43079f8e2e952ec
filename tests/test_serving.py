"""Host side of the serving operators (no GPU): rotary tables, refusals of the C-ABI, workspace sizes."""

import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

from tiktoktechjam2026track3_b200 import _capi, serving
from tiktoktechjam2026track3_b200.build import build

HEADER = Path(__file__).resolve().parents[1] / "include" / "b200tx.h"


@pytest.fixture(scope="module")
def lib():
    build()
    return _capi.load_library()


# ---------------------------------------------------------------------------------- tables
def test_rotary_table_is_the_formula():
    t = serving.rotary_table(50, 32, device="cpu")
    assert t.shape == (50, 16, 2) and t.dtype == torch.float32
    for p in (0, 1, 49):
        for i in (0, 7, 15):
            a = p * 10000.0 ** (-2 * i / 32)
            assert abs(float(t[p, i, 0]) - math.cos(a)) < 1e-7 and abs(float(t[p, i, 1]) - math.sin(a)) < 1e-7


def test_rotary_table_scalings():
    plain = serving.rotary_table(400, 64, device="cpu")
    linear = serving.rotary_table(400, 64, scaling=("linear", 4.0), device="cpu")
    assert torch.equal(linear[::4], plain[:100])  # position 4p turns like p did
    ntk = serving.rotary_table(400, 64, scaling=("ntk", 4.0), device="cpu")
    torch.testing.assert_close(ntk[:, 0], plain[:, 0])  # the fastest pair is unchanged
    torch.testing.assert_close(ntk[::4, -1], plain[:100, -1], atol=1e-6, rtol=0)  # the slowest divided by the factor
    parts = serving.rotary_table(400, 64, scaling=("parts", 4.0, 4096), device="cpu")
    gain = 0.1 * math.log(4.0) + 1.0
    torch.testing.assert_close(parts[:, 0], plain[:, 0] * gain)  # 4096 / 2 pi turns: above 32
    torch.testing.assert_close(parts[::4, -1], plain[:100, -1] * gain)  # less than one turn
    i = 16  # 4096 * 10000^-0.5 / 2 pi = 6.5 turns: on the ramp
    turns = 4096 * 10000.0**-0.5 / (2 * math.pi)
    keep = (turns - 1) / 31
    rate = 10000.0**-0.5 * (keep + (1 - keep) / 4)
    assert abs(float(parts[100, i, 0]) - gain * math.cos(100 * rate)) < 1e-6


@pytest.mark.parametrize("args", [(10, 24), (10, 0), (0, 16), (10, 16, 1.0), (10, 16, 1e4, ("cubic", 2.0)),
                                  (10, 16, 1e4, ("linear", 0.5)), (10, 16, 1e4, ("parts", 2.0, 64, 4, 2))])
def test_rotary_table_refusals(args):
    with pytest.raises(ValueError):
        serving.rotary_table(*args, device="cpu")


# ---------------------------------------------------------------------------------- refusals
P = 256  # addresses that no refused call looks at
ODD = 264


def _call(fn, layout, *args):
    """An entry point that takes its arguments as a struct; None is a null pointer."""
    return fn(layout.pack(*(0 if a is None else a for a in args)), None)


def test_rotary_rejects_bad_arguments(lib):
    def call(x=P, ld_x=128, tokens=4, heads=2, head_dim=64, rotary_dim=64, pos=P, table=P, most=10, out=P, ld_out=128):
        return _call(lib.b2_rotary_fwd, _capi.ROTARY_ARGS, x, ld_x, tokens, heads, head_dim, rotary_dim, 0, 0, pos, table,
                     most, out, ld_out)

    assert call(x=None) == 1 and call(pos=None) == 1 and call(table=None) == 1 and call(out=None) == 1
    assert call(tokens=-1) == 1 and call(heads=0) == 1 and call(most=0) == 1
    assert call(head_dim=24) == 2 and call(head_dim=512, ld_x=1024, ld_out=1024) == 2
    assert call(rotary_dim=80) == 2 and call(rotary_dim=8) == 2 and call(rotary_dim=0) == 2
    assert b"rotary_dim" in lib.b2_last_error()
    assert call(ld_x=120) == 2 and call(ld_out=132) == 2 and call(x=8) == 2
    assert call(tokens=0, x=None) == 0  # empty is a no-op


def _desc(**changes):
    fields = dict(k=256, v=256, k_scale=256, v_scale=256, pages=8, kv_heads=2, page_size=32, head_dim=64,
                  page_stride=2 * 32 * 64, head_stride=32 * 64, dtype=_capi.CACHE_E4M3)
    return _capi.KVCacheDesc(**(fields | changes))


BAD_CACHES = [
    (dict(k=None), 1), (dict(v=None), 1), (dict(k_scale=None), 1), (dict(dtype=7), 1), (dict(pages=0), 1),
    (dict(kv_heads=0), 1), (dict(page_size=24), 2), (dict(page_size=8), 2), (dict(page_size=512), 2),
    (dict(head_dim=40), 2), (dict(page_stride=2 * 32 * 64 - 16), 1), (dict(head_stride=32 * 64 - 16), 1),
    (dict(head_stride=32 * 64 + 8, page_stride=3 * 32 * 64), 2), (dict(k=264), 2),
]


@pytest.mark.parametrize("change,status", BAD_CACHES)
def test_bad_caches_are_rejected(lib, change, status):
    c = _desc(**change)

    def append(cache):
        return _call(lib.b2_cache_append_fwd, _capi.CACHE_APPEND_ARGS, cache, P, 512, 0, 256, 384, 4, 4, 1, P, P, P, P, 2, 4,
                     P, 64, 64, 0, P, 256, None, 0)

    def attend(cache):
        return _call(lib.b2_cache_attention_fwd, _capi.CACHE_ATTENTION_ARGS, cache, P, 256, 1, 1, 4, P, 2, P, 0, 0, 0.125, P,
                     256, P, 1 << 30)

    assert append(ctypes.addressof(c)) == status and attend(ctypes.addressof(c)) == status
    assert append(None) == 1 and attend(None) == 1


def test_a_missing_argument_struct_is_rejected(lib):
    for fn in (lib.b2_rotary_fwd, lib.b2_cache_append_fwd, lib.b2_cache_attention_fwd, lib.b2_window_attention_fwd):
        assert fn(None, None) == 1 and b"null" in lib.b2_last_error()


def test_argument_structs_have_the_headers_layout():
    """Members of each struct in the header, all 8 bytes wide, against what the binding packs."""
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    for name, layout in (("rotary", _capi.ROTARY_ARGS), ("cache_append", _capi.CACHE_APPEND_ARGS),
                         ("cache_attention", _capi.CACHE_ATTENTION_ARGS), ("window_attention", _capi.WINDOW_ATTENTION_ARGS)):
        body = re.search(r"typedef struct b2_%s_args \{(.*?)\}" % name, text, flags=re.S).group(1)
        kinds = ""
        for line in filter(None, (part.strip() for part in body.split(";"))):
            kinds += ("d" if line.startswith("double") else "q") * len(line.split(","))
        packed = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([qd])", layout.format))
        assert kinds == packed, name


def test_cache_append_rejects_bad_arguments(lib):
    def call(qkv=P, ld=512, cols=(0, 256, 384), tokens=4, heads=4, batch=1, start=P, count=P, past=P, pages=P,
             table_pages=2, most=4, table=P, positions=64, rotary_dim=64, q_out=P, ld_q=256, k_out=None, ld_k=0):
        cache = _desc()
        return _call(lib.b2_cache_append_fwd, _capi.CACHE_APPEND_ARGS, ctypes.addressof(cache), qkv, ld, *cols, tokens, heads,
                     batch, start, count, past, pages, table_pages, most, table, positions, rotary_dim, 0, q_out, ld_q, k_out,
                     ld_k)

    for name in ("qkv", "start", "count", "past", "pages", "table", "q_out"):
        assert call(**{name: None}) == 1, name
    assert call(heads=3) == 1 and b"multiple" in lib.b2_last_error()
    assert call(tokens=-1) == 1 and call(batch=-1) == 1 and call(table_pages=0) == 1 and call(positions=0) == 1
    assert call(rotary_dim=24) == 2 and call(rotary_dim=128) == 2
    assert call(cols=(0, 256, 392)) == 1 and call(cols=(4, 256, 384)) == 2 and call(ld=516) == 2
    assert call(ld_q=248) == 2 and call(k_out=P, ld_k=64) == 2 and call(batch=70000) == 2
    assert call(q_out=ODD) == 2
    assert call(tokens=0) == 0 and call(batch=0) == 0 and call(most=0) == 0


def test_cache_attention_rejects_bad_arguments(lib):
    need = _capi.cache_attention_workspace(3, 1, 4, 2, 64, sm_count=148)

    def call(cache=None, q=P, ld_q=256, batch=3, q_len=1, heads=4, pages=P, table_pages=2, kv=P, window=0, sinks=0,
             scale=0.125, out=P, ld_out=256, ws=P, ws_bytes=1 << 30):
        desc = cache or _desc()
        return _call(lib.b2_cache_attention_fwd, _capi.CACHE_ATTENTION_ARGS, ctypes.addressof(desc), q, ld_q, batch, q_len,
                     heads, pages, table_pages, kv, window, sinks, scale, out, ld_out, ws, ws_bytes)

    for name in ("q", "pages", "kv", "out", "ws"):
        assert call(**{name: None}) == 1, name
    assert call(heads=3) == 1 and call(q_len=0) == 1 and call(scale=0.0) == 1 and call(scale=math.nan) == 1
    assert call(window=-1) == 1 and call(sinks=-1) == 1 and call(sinks=4) == 1
    assert call(ld_q=248) == 2 and call(ld_out=260) == 2 and call(ws=ODD) == 2 and call(q=ODD) == 2
    assert call(batch=20000) == 2 and call(table_pages=1 << 40) == 2
    assert call(cache=_desc(head_dim=48, page_stride=4096, head_stride=2048)) == 2
    assert b"head_dim" in lib.b2_last_error()
    assert call(batch=0) == 0
    assert need > 0 and _capi.cache_attention_workspace(6, 1, 4, 2, 64, sm_count=148) >= need
    with pytest.raises(RuntimeError):
        _capi.cache_attention_workspace(3, 1, 5, 2, 64, sm_count=148)


def test_window_attention_rejects_bad_arguments(lib):
    def call(q=P, ld_q=256, k=P, ld_k=128, v=P, ld_v=128, batch=2, seq=100, heads=4, kv_heads=2, head_dim=64, kv_len=None,
             window=10, sinks=2, scale=0.125, out=P, ld_out=256):
        return _call(lib.b2_window_attention_fwd, _capi.WINDOW_ATTENTION_ARGS, q, ld_q, k, ld_k, v, ld_v, batch, seq, heads,
                     kv_heads, head_dim, kv_len, window, sinks, scale, out, ld_out)

    for name in ("q", "k", "v", "out"):
        assert call(**{name: None}) == 1, name
        assert call(**{name: 8}) == 2, name
    assert call(heads=3) == 1 and call(kv_heads=0) == 1 and call(batch=-1) == 1 and call(scale=-1.0) == 1
    assert call(window=-1) == 1 and call(sinks=-1) == 1 and call(window=0) == 1  # sinks without a window
    assert call(head_dim=48) == 2 and call(head_dim=256, ld_q=1024, ld_k=512, ld_v=512, ld_out=1024) == 2
    assert call(ld_q=248) == 1 and call(ld_k=120) == 1 and call(ld_out=257) == 2
    assert call(seq=1 << 40) == 2 and call(batch=70000) == 2
    assert call(batch=0) == 0 and call(seq=0) == 0


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        serving.rotary(x, torch.zeros(4, dtype=torch.int32), serving.rotary_table(8, 64, device="cpu"), 64)
    with pytest.raises(ValueError, match="CUDA"):
        serving.KVCache(torch.zeros(2, 1, 16, 16, dtype=torch.bfloat16), torch.zeros(2, 1, 16, 16, dtype=torch.bfloat16))


def test_streaming_refusals():
    from tiktoktechjam2026track3_b200 import StreamingTransformer, TransformerConfig, UserOptimizedTransformer

    def model(heads=4, causal=True):
        return UserOptimizedTransformer(TransformerConfig(1, 8, 64, heads, 64, 1, causal))

    with pytest.raises(ValueError, match="causal"):
        StreamingTransformer(model(1, causal=False), 1, 8)
    with pytest.raises(NotImplementedError, match="head_dim"):
        StreamingTransformer(model(4), 1, 8)  # head_dim 16
    for bad in (dict(window=-1), dict(sinks=2), dict(window=2, sinks=-1)):
        with pytest.raises(ValueError):
            StreamingTransformer(model(1), 1, 8, **bad)
    with pytest.raises(ValueError, match="table"):
        StreamingTransformer(model(1), 1, 8, table=serving.rotary_table(4, 64, device="cpu"))
    with pytest.raises(RuntimeError, match="GPU"):
        StreamingTransformer(model(1), 1, 8)
