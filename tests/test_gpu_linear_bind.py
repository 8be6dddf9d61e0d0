"""Bound linear_step / linear_extend calls: every layer's operands, decays per
token and per head, host and device slots, the stream of a run."""
from __future__ import annotations

import numpy as np
import pytest

from mitten_amd import STATE_NONE, DeviceStatePool, StateDesc
from mitten_amd import device_pool as dp
from tests.helpers import to_device
from tests.test_gpu_linear import inputs

pytestmark = pytest.mark.gpu

HK, HV, DK, DV, L = 2, 4, 64, 128, 3


def operands(rng, n, layered, head_decay, dtype="bf16"):
    """q, k, v and decays on the device: [L, ...], or without layers."""
    import torch

    per = [[to_device(x) for x in inputs(rng, n, HK, HV, DK, DV, dtype)] for _ in range(L if layered else 1)]
    if head_decay:
        per = [x[:3] + [x[3][0].contiguous()] for x in per]
    return [torch.stack(x) for x in zip(*per)] if layered else per[0]


@pytest.mark.parametrize("layered", [False, True])
@pytest.mark.parametrize("head_decay", [False, True])
@pytest.mark.parametrize("kind", ["step", "step_device", "extend"])
def test_bound_calls_equal_the_unbound(layered, head_decay, kind):
    import torch

    rng = np.random.default_rng(3)
    lens = [70, 0, 33] if kind == "extend" else [1, 1, 1]
    n = sum(lens)
    io = operands(rng, n, layered, head_decay)
    src, dst = np.array([4, STATE_NONE, 2], np.uint32), np.array([1, 3, 2], np.uint32)
    if kind == "step_device":
        src, dst = (torch.from_numpy(x.view(np.int32)).cuda() for x in (src, dst))
    with DeviceStatePool(StateDesc(L, HK, HV, DK, DV, 5, "bf16")) as pool:
        start = torch.randn(pool.desc.shape, device="cuda")
        want = []
        pool.tensor().copy_(start)
        for layer in range(L):
            row = [x[layer] for x in io] if layered else io
            more = (lens,) if kind == "extend" else ()
            want.append((pool.linear_extend if more else pool.linear_step)(layer, *row, *more, dst, src_slots=src))
        states = pool.tensor().clone()
        pool.tensor().copy_(start)
        out = torch.full((L, n, HV, DV) if layered else (n, HV, DV), 7.0, dtype=torch.bfloat16, device="cuda")
        if kind == "extend":
            run = pool.bind_linear_extend(*io, np.array(lens, np.int32), dst, out, src_slots=src)
        else:
            run = pool.bind_linear_step(*io, dst, out, src_slots=src)
        for layer in (2, 0, 1):
            run(layer)
            assert torch.equal(out[layer] if layered else out, want[layer])
            if layered and layer == 2:
                assert bool((out[:2] == 7.0).all())
        assert torch.equal(pool.tensor(), states)
        pool.check()


def test_bind_refusals_and_a_closed_pool():
    import torch

    rng = np.random.default_rng(4)
    io = operands(rng, 3, True, False)
    out = torch.empty_like(io[2])
    pool = DeviceStatePool(StateDesc(L, HK, HV, DK, DV, 5, "bf16"))
    for call, msg in (
        (lambda: pool.bind_linear_step(*(x[:2].contiguous() for x in io), [0, 1, 2], out), "q has shape"),
        (lambda: pool.bind_linear_step(*io, [0, 1], out), "3 rows for 2 slots"),
        (lambda: pool.bind_linear_step(*io, [0, 1, 2], out[:1]), "out has shape"),
        (lambda: pool.bind_linear_extend(*io, [1, 1], [0, 1], out), "add up to 2"),
        (lambda: pool.bind_linear_extend(*io, [1, 2], torch.arange(2, dtype=torch.int32, device="cuda"), out), "host array"),
    ):
        with pytest.raises(dp.BackendError) as ei:
            call()
        assert msg in str(ei.value), (msg, str(ei.value))
    runs = [pool.bind_linear_step(*io, [0, 1, 2], out), pool.bind_linear_extend(*io, [1, 1, 1], [0, 1, 2], out)]
    torch.cuda.synchronize()
    pool.close()
    for run in runs:
        with pytest.raises(dp.BackendError) as ei:
            run(0)
        assert "pool is NULL" in str(ei.value)


def test_a_call_bound_before_a_capture_is_captured():
    """Bound on one stream, run under another and in a graph: every replay
    moves the states on once, and nothing runs outside it."""
    import torch

    rng = np.random.default_rng(5)
    io = operands(rng, 3, True, False)
    out = torch.empty_like(io[2])
    slots = torch.tensor([3, 0, 4], dtype=torch.int32, device="cuda")
    with DeviceStatePool(StateDesc(L, HK, HV, DK, DV, 5, "bf16")) as pool:
        run = pool.bind_linear_step(*io, slots, out)
        start = torch.randn(pool.desc.shape, device="cuda")
        pool.tensor().copy_(start)
        want = []
        for _ in range(3):
            for layer in range(L):
                run(layer)
            torch.cuda.synchronize()
            want.append((out.clone(), pool.tensor().clone()))
        pool.tensor().copy_(start)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for layer in range(L):
                run(layer)
        torch.cuda.synchronize()
        assert torch.equal(pool.tensor(), start)
        for o, s in want:
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, o) and torch.equal(pool.tensor(), s)
        pool.check()


@pytest.mark.parametrize("form", ["step", "step_device", "extend", "extend_device", "bind"])
def test_an_output_over_an_operand_is_refused(form):
    import torch

    n, h, d = 8, 2, 64
    with DeviceStatePool(StateDesc(1, h, h, d, d, n, "f32")) as pool:
        pool.tensor().zero_()
        # q, k, v and room for two outputs one after another; decays in the last of them.
        flat = torch.zeros(5 * n * h * d, device="cuda")
        q, k, v, o, p = (x.view(n, h, d) for x in flat.chunk(5))
        g = p.view(-1)[: n * h].view(n, h)
        slots = torch.arange(n, dtype=torch.int32, device="cuda")
        ip = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        call = {"step": lambda o: pool.linear_step(0, q, k, v, g, list(range(n)), out=o),
                "step_device": lambda o: pool.linear_step(0, q, k, v, g, slots, out=o),
                "extend": lambda o: pool.linear_extend(0, q, k, v, g, [n], [0], out=o),
                "extend_device": lambda o: pool.linear_extend_device(0, q, k, v, g, ip, slots[:1], n, out=o),
                "bind": lambda o: pool.bind_linear_step(q, k, v, g, slots, o)(0)}[form]
        near = [flat[x:x + n * h * d].view(n, h, d) for x in (4, n * h * d - 4, 3 * n * h * d - 4)]
        for bad in (q, k, v, p, *near):
            with pytest.raises(dp.BackendError) as ei:
                call(bad)
            assert "overlaps" in str(ei.value)
        call(o)  # right behind v and before the decays
        pool.check()
