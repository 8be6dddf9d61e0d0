"""What a bound linear_step / linear_extend call hands to the library (CPU:
the library's entry points are replaced by a recorder)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from mitten_amd import STATE_NONE, BackendError, DeviceStatePool, StateDesc, state_pool


class Recorder:
    """Stands in for libmitten_kv: notes the host metadata a call arrives with."""

    def __init__(self):
        self.calls, self.at = [], []

    def mkv_linear_extend_host(self, h, layer, q, k, v, g, o, lens, src, dst, n, scale, flags, stream):
        self.at.append((h, stream))
        self.calls.append((layer, lens[:n], None if not src else src[:n], dst[:n]))
        return 0

    def mkv_linear_step_host(self, h, layer, q, k, v, g, o, src, dst, n, scale, flags, stream):
        self.at.append((h, stream))
        self.calls.append((layer, None, None if not src else src[:n], dst[:n]))
        return 0


@pytest.fixture
def pool(monkeypatch):
    monkeypatch.setattr(state_pool, "_check", lambda *a: None)
    p = DeviceStatePool.__new__(DeviceStatePool)
    p.desc, p.device, p._lib, p._h = StateDesc(2, 1, 2, 64, 64, 9, "f32"), 0, Recorder(), None
    p.stream = type("Stream", (), {"cuda_stream": 0})()
    return p


def rows(n):
    return [torch.zeros(n, h, 64) for h in (1, 1, 2)] + [torch.zeros(n, 2)], torch.zeros(n, 2, 64)


@pytest.mark.parametrize("kind", ["array", "tensor", "list"])
@pytest.mark.parametrize("step", [False, True])
def test_a_bound_call_keeps_its_own_host_arrays(pool, step, kind):
    """Arrays that a caller fills for its next step while a bound call lives
    do not change what that call runs (lengths that it never checked would
    send its kernels past the rows)."""
    make = {"array": lambda x, t: np.array(x, t), "list": lambda x, t: list(x),
            "tensor": lambda x, t: torch.tensor(x, dtype=torch.int64 if t is np.uint32 else torch.int32)}[kind]
    lens = make([2, 1, 4], np.int32)
    src, dst = make([5, STATE_NONE, 7], np.uint32), make([5, 6, 7], np.uint32)
    io, out = rows(3 if step else 7)
    if step:
        run = pool.bind_linear_step(*io, dst, out, src_slots=src, stream=pool.stream)
    else:
        run = pool.bind_linear_extend(*io, lens, dst, out, src_slots=src, stream=pool.stream)
    for x in (lens, src, dst):
        x[0], x[1], x[2] = 1, 2, 3
    run(1)
    assert pool._lib.calls == [(1, None if step else [2, 1, 4], [5, STATE_NONE, 7], [5, 6, 7])]


def test_lists_are_bound_too(pool):
    io, out = rows(3)
    pool.bind_linear_step(*io, [1, 2, 3], out, stream=pool.stream)(0)
    pool.bind_linear_extend(*io, (2, 0, 1), (1, 2, 3), out, stream=pool.stream)(1)
    assert pool._lib.calls == [(0, None, None, [1, 2, 3]), (1, [2, 0, 1], None, [1, 2, 3])]


@pytest.mark.parametrize("step", [False, True])
def test_a_run_takes_the_stream_that_is_current_then(pool, step, monkeypatch):
    """Not the one at the bind: a call bound before a graph's capture must be
    captured with the rest. A given stream stays."""
    now = [11]
    monkeypatch.setattr(state_pool, "_raw_stream", lambda s, device: now[0] if s is None else s.cuda_stream)
    io, out = rows(3)
    bind, more = (pool.bind_linear_step, ()) if step else (pool.bind_linear_extend, ([1, 1, 1],))
    current = bind(*io, *more, [1, 2, 3], out)
    given = bind(*io, *more, [1, 2, 3], out, stream=type("Stream", (), {"cuda_stream": 5})())
    current(0)
    now[0] = 12
    current(1)
    given(1)
    assert [stream for _, stream in pool._lib.at] == [11, 12, 5]


@pytest.mark.parametrize("step", [False, True])
def test_a_run_after_close_has_no_pool(pool, step):
    """The library refuses it (no pool), where it would use freed memory."""
    pool._h = 77
    io, out = rows(3)
    bind, more = (pool.bind_linear_step, ()) if step else (pool.bind_linear_extend, ([1, 1, 1],))
    run = bind(*io, *more, [1, 2, 3], out, stream=pool.stream)
    run(0)
    pool._h = None
    run(0)
    assert [h for h, _ in pool._lib.at] == [77, None]


@pytest.mark.parametrize("step", [False, True])
def test_a_bound_call_needs_out_and_a_layer_of_the_pool(pool, step):
    """(Layer -1 would be the last one of the list of calls.)"""
    io, out = rows(3)
    bind, more = (pool.bind_linear_step, ()) if step else (pool.bind_linear_extend, ([1, 1, 1],))
    with pytest.raises(BackendError):
        bind(*io, *more, [1, 2, 3], None, stream=pool.stream)
    with pytest.raises(BackendError):
        bind(None, *io[1:], *more, [1, 2, 3], out, stream=pool.stream)
    run = bind(*io, *more, [1, 2, 3], out, stream=pool.stream)
    for layer in (-1, 2):
        with pytest.raises(BackendError) as ei:
            run(layer)
        assert f"layer {layer} out of range" in str(ei.value)
    assert not pool._lib.calls
