"""The host side of the per-head operators (afhip_rotary_*, afhip_window_*),
without a GPU: what their descriptors refuse, their workspaces, and the
rotation's frequencies."""
import ctypes
import math

import numpy as np
import pytest


def window(**change):
    from afhip import _lib

    d = dict(batch=2, queries=5, keys=70, query_heads=4, key_heads=2, head_dim=64, left=8, right=0, sinks=2,
             dtype=_lib.F16, scale=0.125)
    strides = {n: change.pop(n) for n in ("q", "k", "v", "out") if n in change}
    desc = _lib.WindowDesc(**{**d, **change})
    for name, s in strides.items():
        setattr(desc, name, _lib.Strides(*s))
    return desc


def rotary(**change):
    from afhip import _lib

    d = dict(batch=2, tokens=5, query_heads=4, key_heads=2, head_dim=64, rotary_dim=32, layout=0, norm=1,
             dtype=_lib.F16, capacity=0, epsilon=1e-5, rotation_scale=1.0)
    strides = {n: change.pop(n) for n in ("q", "k") if n in change}
    desc = _lib.RotaryDesc(**{**d, **change})
    for name, s in strides.items():
        setattr(desc, name, _lib.Strides(*s))
    return desc


def size(name, desc):
    from afhip import _lib

    bytes_ = ctypes.c_size_t()
    _lib.call(name, ctypes.byref(desc), ctypes.byref(bytes_))
    return bytes_.value


@pytest.mark.parametrize("change, message", [
    (dict(batch=0), "positive"), (dict(queries=0), "positive"), (dict(keys=0), "positive"),
    (dict(head_dim=-8), "positive"), (dict(head_dim=12), "multiple of 8"), (dict(head_dim=136), "multiple of 8"),
    (dict(query_heads=5), "5 query heads over 2"), (dict(left=-2), "at least -1"), (dict(right=-2), "at least -1"),
    (dict(sinks=-1), "at least"), (dict(dtype=2), "f32 or f16"), (dict(scale=0.0), "positive and finite"),
    (dict(scale=-1.0), "positive and finite"), (dict(scale=math.nan), "positive and finite"),
    (dict(scale=math.inf), "positive and finite"), (dict(keys=1 << 30), "2\\^30"),
    (dict(queries=1 << 29), "2\\^30"),
    (dict(k=(70 * 128, 128, -64)), "negative stride"), (dict(k=(70 * 128, 132, 64)), "16 bytes"),
    (dict(v=(70 * 128, 1 << 24, 64)), "16 MiB"), (dict(k=(70 * 128, 32, 64)), "tokens that overlap"),
    (dict(out=(5 * 256, 256, 0)), "entries that overlap"), (dict(out=(0, 256, 64)), "entries that overlap"),
    (dict(out=(5 * 256, 64, 64)), "entries that overlap"), (dict(out=(5 * 256 - 8, 256, 64)), "entries that overlap"),
    (dict(q=(1 << 50, 256, 64)), "too large"),
])
def test_window_refusals(change, message):
    from afhip import _lib

    for name in ("afhip_window_workspace_size", "afhip_window_backward_workspace_size"):
        with pytest.raises(_lib.RangeError, match=message):
            size(name, window(**change))


@pytest.mark.parametrize("change, message", [
    (dict(batch=0), "positive"), (dict(tokens=-1), "positive"), (dict(key_heads=0), "positive"),
    (dict(head_dim=20), "multiple of 8"), (dict(head_dim=256), "multiple of 8"),
    (dict(rotary_dim=10), "multiple of 4"), (dict(rotary_dim=72), "multiple of 4"), (dict(rotary_dim=-8), "multiple"),
    (dict(layout=2), "layout"), (dict(norm=3), "norm"), (dict(dtype=2), "f32 or f16"), (dict(capacity=-1), "capacity"),
    (dict(epsilon=-1.0), "epsilon"), (dict(epsilon=math.nan), "epsilon"), (dict(rotation_scale=math.inf), "finite"),
    (dict(batch=1 << 20, tokens=1 << 10), "2\\^29"), (dict(q=(5 * 256, 256, 4)), "16 bytes"),
    (dict(k=(5 * 128, 32, 64)), "tokens that overlap"),
])
def test_rotary_refusals(change, message):
    from afhip import _lib

    with pytest.raises(_lib.RangeError, match=message):
        size("afhip_rotary_backward_workspace_size", rotary(**change))


def test_repeated_entries_are_taken():
    # One batch entry's or head's keys for all: a stride of 0, for inputs.
    assert size("afhip_window_workspace_size", window(k=(0, 128, 64), v=(0, 128, 0))) == 0
    size("afhip_rotary_backward_workspace_size", rotary(q=(0, 256, 0)))


def test_written_strides_in_any_order():
    # Heads outside the tokens, and rows with gaps.
    size("afhip_window_workspace_size", window(out=(4 * 5 * 64, 64, 5 * 64)))
    size("afhip_window_workspace_size", window(out=(64, 2 * 4 * 64, 2 * 64)))
    size("afhip_window_workspace_size", window(out=(5 * 1000, 1000, 72)))


def test_workspaces():
    # Short spans need none; one query over a long cache is split, each part a row of head_dim sums and two more f32.
    assert size("afhip_window_workspace_size", window()) == 0
    long = window(batch=1, queries=1, keys=40000, left=-1)
    row = 4 * (64 + 2) * 4
    assert size("afhip_window_workspace_size", long) % row == 0
    assert 2 <= size("afhip_window_workspace_size", long) // row <= 64
    # A window bounds the span whatever the cache holds.
    assert size("afhip_window_workspace_size", window(batch=1, queries=1, keys=40000, left=100)) == 0
    # The way back keeps 16 bytes a row.
    assert size("afhip_window_backward_workspace_size", window()) >= 2 * 5 * 4 * 16
    # Only tiles of keys that every row sees, here those of the sinks, are cut into chunks of rows: 16 bytes a row, and
    # the sums of two tiles of 128 keys in at most 64 chunks.
    long = dict(batch=1, queries=131072, keys=131072, query_heads=32, key_heads=8, head_dim=128, left=1023)
    rows = 131072 * 32 * 16
    assert size("afhip_window_backward_workspace_size", window(**long, sinks=0)) == rows
    sinks = size("afhip_window_backward_workspace_size", window(**long, sinks=200))
    assert rows < sinks <= rows + 8 * 2 * 64 * 2 * 128 * 128 * 4
    assert size("afhip_rotary_backward_workspace_size", rotary(norm=0)) == 0
    assert size("afhip_rotary_backward_workspace_size", rotary(norm=2)) > 0


def test_runs_need_the_device():
    from afhip import _lib

    lib = _lib.library()
    none = [None] * 20
    assert lib.afhip_rotary_run(ctypes.byref(rotary()), *none[:15]) == _lib.ERR_NOT_OPEN
    assert lib.afhip_rotary_backward(ctypes.byref(rotary()), *none[:17], 0, None) == _lib.ERR_NOT_OPEN
    assert lib.afhip_window_run(ctypes.byref(window()), *none[:8], 0, None) == _lib.ERR_NOT_OPEN
    assert lib.afhip_window_backward(ctypes.byref(window()), *none[:6], None, *none[:6], 0, None) == _lib.ERR_NOT_OPEN
    for name in ("afhip_window_workspace_size", "afhip_window_backward_workspace_size",
                 "afhip_rotary_backward_workspace_size"):
        assert getattr(lib, name)(None, None) == _lib.ERR_INVALID_ARGUMENT


def test_frequencies():
    from afhip import _lib, rotary as op

    plain = op.frequencies(64, base=1000.0)
    assert plain.dtype == np.float64 and plain.shape == (32,)
    assert plain[0] == 1.0 and np.allclose(plain, 1000.0 ** (-np.arange(32) / 32), rtol=1e-15)
    assert np.array_equal(op.frequencies(64, base=1000.0, scaling="linear", factor=4.0), plain / 4)
    ntk = op.frequencies(64, base=1000.0, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], plain[-1] / 4, rel_tol=1e-12)
    yarn = op.frequencies(64, base=1000.0, scaling="yarn", factor=4.0, trained_length=2048)
    turns = 2048 * plain / (2 * math.pi)
    assert np.array_equal(yarn[turns >= 32], plain[turns >= 32])
    assert np.allclose(yarn[turns <= 1], plain[turns <= 1] / 4, rtol=1e-15)
    assert (yarn <= plain).all() and (yarn >= plain / 4).all()
    assert op.yarn_scale(1.0) == 1.0 and math.isclose(op.yarn_scale(4.0), 0.1 * math.log(4) + 1)
    for bad in (dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=8, scaling="other"),
                dict(rotary_dim=8, factor=0.0), dict(rotary_dim=8, base=-1.0),
                dict(rotary_dim=8, scaling="yarn", fast=1.0, slow=2.0)):
        with pytest.raises(_lib.RangeError):
            op.frequencies(**bad)
