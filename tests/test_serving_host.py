"""What the serving operators' Python side decides before a launch (no GPU)."""

import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

from tiktoktechjam2026track3_b200 import _capi, serving
from tiktoktechjam2026track3_b200.build import build


class _Queries:
    """Stands for q: [rows, width] on the GPU."""

    device = torch.device("cuda", 0)

    def __init__(self, rows, width):
        self.shape = (rows, width)

    def dim(self):
        return 2

    def size(self, i):
        return self.shape[i]


def _cache(monkeypatch, capturing):
    """A cache without tensors whose workspaces are plain lists, on stream 7."""
    cache = object.__new__(serving.KVCache)
    cache.head_dim, cache._workspaces, cache._desc = 64, {}, _capi.KVCacheDesc()
    monkeypatch.setattr(_capi, "_current_device", lambda: 0)
    monkeypatch.setattr(_capi, "_stream_of", lambda device: 7)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    monkeypatch.setattr(cache, "workspace", lambda *size: list(size), raising=False)
    return cache


def test_a_captured_call_has_a_workspace_of_its_own(monkeypatch):
    """A graph may outlive the workspace that its stream keeps, and run next to the stream's other calls."""
    capturing = [False]
    cache = _cache(monkeypatch, capturing)
    kept = cache._workspace(_Queries(2, 256), 1)
    assert cache._workspace(_Queries(1, 256), 1) is kept  # smaller calls of the stream share it
    capturing[0] = True
    first, second = cache._workspace(_Queries(2, 256), 1), cache._workspace(_Queries(2, 256), 1)
    assert first is not kept and second is not kept and first is not second
    larger = cache._workspace(_Queries(64, 256), 1)
    assert all(larger is not w for _, w in cache._workspaces.values())
    capturing[0] = False
    assert cache._workspace(_Queries(2, 256), 1) is kept


def test_cache_attention_reads_its_pages_past_the_read_only_path():
    """The launch that writes pages and scales may still run when the attention's first CTAs are resident."""
    text = (Path(serving.__file__).parent / "csrc" / "cache_attention.cuh").read_text()
    assert "pdl_wait_previous_grid" in text
    assert not re.search(r"__ldg|ld\.global(\.\w+)*\.nc", text)


@pytest.mark.parametrize("head_dim", [32, 64, 128])
def test_workspace_does_not_grow_with_the_row_blocks(head_dim):
    """512 rows to a key head (32 blocks of 16) at a time; more take turns."""
    build()

    def size(q_len, heads, batch=4):
        return _capi.cache_attention_workspace(batch, q_len, heads, 8, head_dim, sm_count=148)

    assert size(1, 8) <= size(2, 64) < size(4, 64) < size(64, 64) == size(1024, 64) <= 161_000_000


def test_workspace_is_alike_for_every_batch():
    """Its counters lie at one place for every call: a workspace is either too small, and refused, or right."""
    build()
    sizes = {_capi.cache_attention_workspace(batch, 2, 4 * kv, kv, 64, sm_count=148) for batch in (1, 64, 4096) for kv in (1, 8)}
    assert len(sizes) == 1


# ---------------------------------------------------------------------------------- arguments at their types' ends
HUGE, P = (1 << 63) - 8, 256  # a multiple of 8; an address that nobody looks at: the calls have no rows


def _refused(lib, entry, layout, args):
    """Whether a call without rows, which does nothing if it passes the checks, is refused."""
    status = getattr(lib, entry)(layout.pack(*args), None)
    assert status in (0, 1, 2)
    return status != 0


def _desc(**changes):
    fields = dict(k=256, v=256, k_scale=256, v_scale=256, pages=8, kv_heads=5, page_size=32, head_dim=64,
                  page_stride=5 * 32 * 64, head_stride=32 * 64, dtype=_capi.CACHE_E4M3)
    return _capi.KVCacheDesc(**(fields | changes))


def _append_args(cache, ld=1024, cols=(0, 320, 640), heads=5, table_pages=2, most=4):
    return (ctypes.addressof(cache), P, ld, *cols, 0, heads, 1, P, P, P, P, table_pages, most, P, 64, 64, 0, P, 320, 0, 0)


def _attend_args(cache, heads=5, q_len=1, table_pages=2, scale=0.125):
    return (ctypes.addressof(cache), P, 320, 0, q_len, heads, P, table_pages, P, 0, 0, scale, P, 320, P, 1 << 30)


def test_sums_and_products_of_arguments_do_not_wrap():
    """Strides, columns and counts near 2^63, whose sums and products with a head's size would look small."""
    build()
    lib = _capi.load_library()
    good = _desc()
    assert not _refused(lib, "b2_cache_append_fwd", _capi.CACHE_APPEND_ARGS, _append_args(good))
    assert not _refused(lib, "b2_cache_attention_fwd", _capi.CACHE_ATTENTION_ARGS, _attend_args(good))
    for bad in (dict(head_stride=1 << 62), dict(head_stride=(1 << 62) + 32 * 64), dict(page_stride=-(1 << 63))):
        cache = _desc(**bad)
        assert _refused(lib, "b2_cache_append_fwd", _capi.CACHE_APPEND_ARGS, _append_args(cache)), bad
        assert _refused(lib, "b2_cache_attention_fwd", _capi.CACHE_ATTENTION_ARGS, _attend_args(cache)), bad
    for bad in (dict(cols=(HUGE, 320, 640)), dict(cols=(0, HUGE, 640)), dict(cols=(0, 320, HUGE)), dict(ld=-(1 << 63)),
                dict(ld=HUGE), dict(heads=5 << 58), dict(table_pages=1 << 60), dict(most=HUGE)):
        assert _refused(lib, "b2_cache_append_fwd", _capi.CACHE_APPEND_ARGS, _append_args(good, **bad)), bad
    for bad in (dict(heads=5 << 58), dict(q_len=1 << 62), dict(table_pages=(1 << 60) - 4),
                dict(scale=math.inf), dict(scale=1e300), dict(scale=1e-300)):
        assert _refused(lib, "b2_cache_attention_fwd", _capi.CACHE_ATTENTION_ARGS, _attend_args(good, **bad)), bad
    for heads, scale in ((1 << 58, 0.125), (1 << 62, 0.125), (1, math.inf)):
        args = (P, 64, P, 64, P, 64, 0, 5, heads, 1, 64, 0, 0, 0, scale, P, 64)
        assert _refused(lib, "b2_window_attention_fwd", _capi.WINDOW_ATTENTION_ARGS, args)
    for args in ((1, 1 << 62, 8, 8, 64), (1, 1, 1 << 62, 1, 64), (1, 1, 8, 8, 48), (1, 1, 8, 8, HUGE)):
        with pytest.raises(RuntimeError):
            _capi.cache_attention_workspace(*args, sm_count=148)
    with pytest.raises(RuntimeError):
        _capi.cache_attention_workspace(1, 1, 8, 8, 64, sm_count=1 << 30)


# ---------------------------------------------------------------------------------- where tensors lie
class _On:
    """What a wrapper asks of a contiguous CUDA tensor, on a device that need not be there."""

    is_cuda = True

    def __init__(self, device, shape, dtype=torch.bfloat16):
        self.device, self.shape, self.dtype = torch.device("cuda", device), tuple(shape), dtype

    def size(self, i=None):
        return self.shape if i is None else self.shape[i]

    def stride(self):
        return tuple(math.prod(self.shape[i + 1:]) for i in range(len(self.shape)))

    def dim(self):
        return len(self.shape)

    def numel(self):
        return math.prod(self.shape)

    def get_device(self):
        return self.device.index

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 256


class _Library:
    """Takes every entry point and keeps (its name, the device that was current, the stream)."""

    def __init__(self, current):
        self.calls, self._current = [], current

    def __getattr__(self, name):
        def entry(args, stream):
            self.calls.append((name, self._current[0], stream))
            return 0
        return entry


@pytest.fixture
def library(monkeypatch):
    current = [0]

    class Device:
        def __init__(self, device):
            self.index = device if isinstance(device, int) else device.index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    fake = _Library(current)
    monkeypatch.setattr(_capi, "_lib", fake)
    monkeypatch.setattr(_capi, "_raw_stream", lambda device: 100 + device)
    monkeypatch.setattr(_capi, "_current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    return fake


def _calls(device):
    """name -> (wrapper, its tensors on `device`, its other arguments)."""
    i32 = torch.int32
    desc = _capi.KVCacheDesc(pages=4, kv_heads=2, page_size=16, head_dim=64)
    desc.device = device

    def on(*shape, dtype=torch.bfloat16):
        return _On(device, shape, dtype)

    return {
        "b2_rotary_fwd": (_capi.rotary, dict(
            x=on(4, 128), positions=on(4, dtype=i32), table=on(9, 32, 2, dtype=torch.float32), out=on(4, 128)),
            dict(head_dim=64)),
        "b2_cache_append_fwd": (_capi.cache_append, dict(
            qkv=on(4, 512), new_start=on(2, dtype=i32), new_len=on(2, dtype=i32), past_len=on(2, dtype=i32),
            page_table=on(2, 3, dtype=i32), table=on(9, 32, 2, dtype=torch.float32), q_out=on(4, 256), k_out=on(4, 128)),
            dict(cache=desc, num_heads=4, q_col=0, k_col=256, v_col=384, max_new=2)),
        "b2_cache_attention_fwd": (_capi.cache_attention, dict(
            q=on(2, 256), page_table=on(2, 3, dtype=i32), kv_len=on(2, dtype=i32), out=on(2, 256),
            workspace=on(1 << 20, dtype=torch.uint8)), dict(cache=desc, q_len=1, window=0, sinks=0, scale=0.1)),
        "b2_window_attention_fwd": (_capi.window_attention, dict(
            q=on(6, 256), k=on(6, 128), v=on(6, 128), kv_len=on(2, dtype=i32), out=on(6, 256)),
            dict(batch=2, seq_len=3, head_dim=64, window=0, sinks=0, scale=0.1)),
    }


@pytest.mark.parametrize("device", [0, 1])
def test_calls_run_on_the_gpu_of_their_tensors(library, device):
    for name, (call, tensors, rest) in _calls(device).items():
        call(**tensors, **rest)
        assert library.calls.pop() == (name, device, 100 + device)
    assert _capi._current_device() == 0


def test_tensors_of_another_gpu_are_refused(library):
    for call, tensors, rest in _calls(0).values():
        for name, t in tensors.items():
            with pytest.raises(ValueError, match="must be on cuda"):
                call(**(tensors | {name: _On(1, t.shape, t.dtype)}), **rest)
    assert not library.calls


# ---------------------------------------------------------------------------------- refusals by type
@pytest.mark.parametrize("scaling", [("ntk",), ("linear", 2.0, 3.0), ("parts", 2.0), ("parts", 2.0, 64, 1.0),
                                     ("parts", 2.0, 0), ("parts", 2.0, 64, 1.0, 32.0, 5.0)])
def test_malformed_scalings_are_value_errors(scaling):
    with pytest.raises(ValueError):
        serving.rotary_table(8, 16, scaling=scaling, device="cpu")


def test_attend_refuses_q_of_another_shape_before_it_makes_a_workspace(monkeypatch):
    cache = _cache(monkeypatch, [False])
    for q, q_len in ((_On(0, (4, 256)), 0), (_On(0, (4, 256)), -1), (_On(0, (256,)), 1), (_On(0, (2, 2, 64)), 1)):
        with pytest.raises(ValueError, match="q must be"):
            serving.KVCache.attend(cache, q, None, None, q_len=q_len, scale=0.1, out=q)
    assert not cache._workspaces


def test_numbers_that_are_not_integers_are_type_errors(library):
    for call, tensors, rest in _calls(0).values():
        for name in {"window", "sinks", "max_new", "q_col"} & set(rest):
            with pytest.raises(TypeError, match="integers"):
                call(**tensors, **(rest | {name: 4.0}))
            with pytest.raises(TypeError, match="integers"):
                call(**tensors, **(rest | {name: 1 << 70}))
    assert not library.calls


def test_heads_of_no_width_are_value_errors(library):
    for name in ("b2_rotary_fwd", "b2_window_attention_fwd"):
        call, tensors, rest = _calls(0)[name]
        for head_dim in (0, -64):
            with pytest.raises(ValueError, match="heads"):
                call(**tensors, **(rest | dict(head_dim=head_dim)))
    assert not library.calls
